// What the tcgen05 kernels over a paged cache share: operand layouts, products, tensor memory accesses, pairs of fp32, the list of a CTA's key tiles.
#pragma once
#include "varq_attn_tc.cuh"
#include "varq_paged.cuh"

namespace varq {
namespace {

constexpr int PT_M = 128, PT_N = 64;

// 16-byte chunk `ch` (eight head_dim values) of row `r` in a 128B-swizzled tile of ROWS rows: blocks of 64 columns
template <int ROWS> __device__ __forceinline__ uint32_t pt_chunk(int r, int ch) {
    return (uint32_t)((ch >> 3) * (ROWS * 128) + (r >> 3) * 1024 + (r & 7) * 128 + (((ch & 7) ^ (r & 7)) << 4));
}
// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void tc_mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// pairs of fp32 in one 64-bit register
using pair = unsigned long long;
__device__ __forceinline__ pair pair_of(float x, float y) { pair d; asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y)); return d; }
__device__ __forceinline__ float pair_x(pair p) { float x; [[maybe_unused]] float y; asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p)); return x; }
__device__ __forceinline__ float pair_y(pair p) { [[maybe_unused]] float x; float y; asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p)); return y; }
__device__ __forceinline__ pair fma2(pair a, pair b, pair c) { pair d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }
__device__ __forceinline__ pair add2(pair a, pair b) { pair d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ pair mul2(pair a, pair b) { pair d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
// 16 rows x 32 columns: thread (g, c) = (lane / 4, lane % 4) gets columns 2c, 2c + 1 of every eight, of row g (r[4n], r[4n + 1]) and row g + 8
__device__ __forceinline__ void tmem_ld_16x256(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
// 16 rows x 16 columns: column c of every four, of row g (r[2n]) and row g + 8 (r[2n + 1])
__device__ __forceinline__ void tmem_st_16x128(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
// waits for the loads from tensor memory in flight, and keeps the use of what they left in `r` behind that
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                   "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
                   "+r"(r[31])
                 :: "memory");
}
__device__ __forceinline__ pair pair_of_bits(uint32_t x, uint32_t y) { pair d; asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(x), "r"(y)); return d; }
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// one arrival for a warp, behind what all its lanes did
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}
template <int BITS> __host__ __device__ constexpr uint32_t pt_neg_base(int cls) {      // fp16 pairs of -(1024 / 2^p + bias), by class of bit position
    return BITS == 8 ? 0xE480E480u : BITS == 4 ? (cls == 0 ? 0xE408E408u : 0xD480D480u)
                                               : (cls == 0 ? 0xE402E402u : cls == 1 ? 0xDC08DC08u : cls == 2 ? 0xD420D420u : 0xCC80CC80u);
}

// The key tiles of a CTA: `ns` tiles of first tokens, then those from `lo` on; `first`: the first key of its windows, in the tile at `lo`
struct PtTiles {
    int ns, lo, n, first;
    __device__ __forceinline__ int key(int i) const { return i < ns ? i * PT_N : lo + (i - ns) * PT_N; }
};

// one of the two 16-element halves of a query row's 32, packed fp16 in element order -> operand order of codes of `kb` bits
__device__ __forceinline__ void q_operand_order(uint32_t (&w)[8], int kb) {
    if (kb == 8) return;
    uint32_t o[8];
    if (kb == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                o[4 * i + 2 * j] = __byte_perm(w[4 * i + j], w[4 * i + 2 + j], 0x5410);
                o[4 * i + 2 * j + 1] = __byte_perm(w[4 * i + j], w[4 * i + 2 + j], 0x7632);
            }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) { o[2 * j] = __byte_perm(w[j], w[4 + j], 0x5410); o[2 * j + 1] = __byte_perm(w[j], w[4 + j], 0x7632); }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = o[i];
}

}  // namespace
}  // namespace varq
