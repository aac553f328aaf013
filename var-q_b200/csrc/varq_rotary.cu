// Norms of queries and keys per head and the rotation by position, in one pass: on their own (varq_rotate), and in front of a paged cache, where the
// rotated keys are quantized straight into their slots (varq_paged_append_rotated).
//
//   x <- x / max(|x|_2, eps)  or  x / sqrt(mean x^2 + eps)  or  x;   x <- x w;   (a, b) <- (a cos t - b sin t, b cos t + a sin t)
//
// for pairs (a, b) of neighbours or of elements half the rotary dimension apart, t = position on the pair's axis times its frequency.
// Angles: a frequency is held as turns per position, a fraction of 64 bits; position times that, modulo 2^64, is the angle in turns with an error of
// position * 2^-65 turns (a product in fp32 is off by whole radians from 10^7 on).  Its upper 32 bits (2^-32 turns more), rounded to fp32 (2^-26 turns), go to sincospi.
// Everything behind is fp32, rounded once to the output's type, or to the code of the cache.
//
// D / 16 neighbouring lanes hold a row with two pieces of eight values each, chosen so that both values of a pair are in one lane.  The lanes of a
// token share its angles, which the block computes once for all heads.  The next rows' pieces are on their way to shared memory (cp.async), three ahead, which keeps enough
// bytes in flight without registers for them.
//
// What bounds it (B200): its bytes, as long as it only turns.  16384 tokens of 16 + 16 heads x 128, bf16, L2 norm: 268 MB in 46 us, 5.8 TB/s (41 us at the copy rate).  In front
// of a cache no unit is full (issue 58 %, DRAM 46 %, 16 warps on an SM): 16384 tokens of 32 + 8 + 8 heads, K in 8 bits, V in 4: 82 us, 55 by its bytes; some 260 instructions
// of a warp for its four rows, where quantized rows take twice those of a query's.  A few tokens: a launch, 3.5 us for 16.  16 bits to fp32 (the first case, in front of an image
// schedule): 403 MB in 74 us, 61 at the copy rate; its 80 registers spill.
// On the way (first case / append; without the test for rows of extreme sizes): values one by one in registers, one row ahead 72 / 111 us; pairs of fp32 in one instruction
// 53 / 111; rows copied ahead 46 / 109; a loop for each of q, k and v, with addresses by steps 46 / 89; registers for two blocks on an SM instead of three where rows are
// quantized 46 / 82; two conversions in an instruction, one factor for a row 45 / 82; blocks of 128 threads 45 / 80.  fp32 rows, whose pieces such copies would take half a
// sector at a time, are held one ahead: 34.8 us for 8192 tokens of 16 + 4 heads (25.6 by its bytes), 44 with copies.
#include <cstring>
#include <type_traits>

#include "varq_paged_rows.cuh"

namespace varq {
namespace {

// Where rows are quantized, 126 registers are needed and smaller blocks begin and end less at a time: 80.0 us against 82.4 with two of 256
template <bool PAGED> constexpr int ROT_THREADS = PAGED ? 128 : 256;

struct RotArgs {
    const unsigned long long* turns; const int32_t* axis; const void* pos;
    int pos_bytes, n_axes, R, inter;
    long long ps_a, ps_b, ps_l;
    int norm; float inv_eps, least, sum_mul, sum_add;      // 1 / sqrt(sum * sum_mul + sum_add), or inv_eps where that sum is less than `least`
    uint32_t fair, fair_span;         // sums of squares of ordinary rows: from 2^-80 and `least` to 2^80 (bits of the first, how far to the last)
    const float *qw, *kw; long long qw_h, qw_d, kw_h, kw_d; int qw_vec, kw_vec;
    const void *q, *k, *v; long long qs_b, qs_l, qs_h, ks_b, ks_l, ks_h, vs_l, vs_h;
    void *qo, *ko; long long qo_b, qo_l, qo_h, ko_b, ko_l, ko_h;
    int Hq, Hk, Hv;
    uint32_t tokens; FastDiv L, half;
    int lanes_log2, parts;            // rows of a token that a block works on side by side (log2), parts of a token's rows
    PagedView c; const long long* slots; float qeps;
};

// pairs of fp32 in one 64-bit register
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float x, float y) { f32x2 d; asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y)); return d; }
__device__ __forceinline__ float2 unpack2(f32x2 p) { float2 v; asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p)); return v; }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { f32x2 d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { f32x2 d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }

// A lane's sixteen values as eight pairs (x[j], y[j]) that turn together, two of them in a register: the pieces themselves where pairs are half the rotary
// dimension apart, even and odd elements where they are neighbours.  Element i of piece e is value `at` of x (or y).
template <bool INTER> struct Pairs {
    f32x2 x[4], y[4];
    __device__ __forceinline__ Pairs(const float (&v)[2][8]) {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            if constexpr (INTER) {
                const float* p = v[m >> 1] + 4 * (m & 1);
                x[m] = pack2(p[0], p[2]); y[m] = pack2(p[1], p[3]);
            } else {
                x[m] = pack2(v[0][2 * m], v[0][2 * m + 1]); y[m] = pack2(v[1][2 * m], v[1][2 * m + 1]);
            }
        }
    }
    __device__ __forceinline__ void values(float (&v)[2][8]) const {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const float2 a = unpack2(x[m]), b = unpack2(y[m]);
            if constexpr (INTER) {
                float* p = v[m >> 1] + 4 * (m & 1);
                p[0] = a.x; p[1] = b.x; p[2] = a.y; p[3] = b.y;
            } else {
                v[0][2 * m] = a.x; v[0][2 * m + 1] = a.y; v[1][2 * m] = b.x; v[1][2 * m + 1] = b.y;
            }
        }
    }
};

__device__ __forceinline__ float max_abs(float m, float x) {      // a NaN stays one
    float d;
    asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %2;\n\tmax.NaN.f32 %0, %1, t;\n\t}" : "=f"(d) : "f"(m), "f"(x));
    return d;
}

constexpr int ROT_AHEAD = 4;           // places of a thread's ring
__device__ __forceinline__ float rsqrt_normal(float x) {          // of a normal number, an infinity or a NaN
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// eight values, rounded once; two conversions in an instruction
template <typename O, bool VEC> __device__ __forceinline__ void store_piece(O* p, const float (&v)[8]) {
    if constexpr (sizeof(O) == 4 || !VEC) store_vals<O, 8, VEC>(p, v, 8);
    else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<O, __half>::value) { const __half2 x = __floats2half2_rn(v[2 * i], v[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&x); }
            else { const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&x); }
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

enum Role : int { ROLE_Q, ROLE_K, ROLE_V };
template <int V> struct IsRole { static constexpr int value = V; };

template <typename T, typename O, int D, bool VEC, bool PAGED, bool INTER>
__global__ void __launch_bounds__(ROT_THREADS<PAGED>, PAGED ? 4 : sizeof(T) == 4 ? 2 : 3) rotary_kernel(RotArgs a) {
    constexpr int LPR = D / 16, GROUPS = ROT_THREADS<PAGED> / LPR;
    constexpr bool RING = VEC && sizeof(T) == 2;
    extern __shared__ __align__(16) float2 s_cs[];           // [token][pair]: cos, sin
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & (LPR - 1), group = threadIdx.x / LPR, side = 1 << a.lanes_log2;
    const int tb = GROUPS >> a.lanes_log2, half = a.R >> 1;
    const uint32_t block = blockIdx.x / (uint32_t)a.parts, part = blockIdx.x - block * (uint32_t)a.parts;
    const uint32_t t0 = block * tb, t = t0 + (uint32_t)(group >> a.lanes_log2);
    const bool token_there = t < a.tokens;
    const uint32_t b = token_there ? a.L.div(t) : 0, l = token_there ? t - b * a.L.d : 0;
    const int step = side * a.parts, k_row = a.Hq, v_row = a.Hq + a.Hk, end = token_there ? v_row + a.Hv : 0;
    // pieces of a lane: 8 values each, from c0 * 8 and c1 * 8 on
    const int r16 = a.R >> 4;
    const int c0 = INTER || lane < r16 ? lane : 2 * lane, c1 = INTER ? lane + LPR : lane < r16 ? lane + r16 : 2 * lane + 1, apart = (c1 - c0) * 8;
    // the rows of a lane group, one after another: h = first, first + step, ...; where a row is, by steps while it stays one of q, k or v
    auto row_at = [&](int h) -> const T* {
        if (h < k_row) return reinterpret_cast<const T*>(a.q) + b * a.qs_b + l * a.qs_l + h * a.qs_h + c0 * 8;
        if (h < v_row) return reinterpret_cast<const T*>(a.k) + b * a.ks_b + l * a.ks_l + (h - k_row) * a.ks_h + c0 * 8;
        return reinterpret_cast<const T*>(a.v) + l * a.vs_l + (h - v_row) * a.vs_h + c0 * 8;
    };
    int h = (int)part * side + (group & (side - 1)), ahead = h, ahead_end = 0, stage = 0, ahead_stage = 0;
    const T* next = nullptr;
    long long next_step = 0;
    // A thread's pieces of its next rows wait in shared memory, in places that only this thread writes and reads: several rows in flight without their registers.
    // (fp32 rows, of whose pieces such a copy takes half sectors, and rows that are not 16-byte aligned are held in registers, one ahead.)
    unsigned char* const ring = reinterpret_cast<unsigned char*>(s_cs + tb * half) + threadIdx.x * 16;
    constexpr int STAGE = 2 * ROT_THREADS<PAGED> * 16;
    Piece<T, VEC> held[2];
    auto advance = [&]() {                                   // `next`: row `ahead`
        next += next_step;
        if (ahead < ahead_end || ahead >= end) return;
        next = row_at(ahead);
        next_step = step * (ahead < k_row ? a.qs_h : ahead < v_row ? a.ks_h : a.vs_h);
        ahead_end = ahead < k_row ? k_row : ahead < v_row ? v_row : end;
    };
    auto request = [&]() {
        advance();
        if constexpr (RING) {
            if (ahead < end) {
                const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring + ahead_stage);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(next) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + ROT_THREADS<PAGED> * 16), "l"(next + apart) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            ahead_stage = ahead_stage == (ROT_AHEAD - 1) * STAGE ? 0 : ahead_stage + STAGE;
        } else if (ahead < end) {
            held[0].load(next);
            held[1].load(next + apart);
        }
        ahead += step;
    };
#pragma unroll
    for (int i = 0; i < (RING ? ROT_AHEAD - 1 : 1); ++i) request();
    long long slot = -1;
    if (PAGED && token_there) slot = __ldg(a.slots + t);
    const bool kept = PAGED && (unsigned long long)slot < ((unsigned long long)a.c.n_pages << a.c.page_shift);

    // ---- angles of the block's tokens
    for (int i = threadIdx.x; i < tb * half; i += ROT_THREADS<PAGED>) {
        const int tk = (int)a.half.div((uint32_t)i), p = i - tk * half;
        const uint32_t tt = t0 + tk;
        float s = 0.f, c = 1.f;
        if (tt < a.tokens) {
            const uint32_t bb = a.L.div(tt), ll = tt - bb * a.L.d;
            const int ax = min(max(__ldg(a.axis + p), 0), a.n_axes - 1);
            const long long at = ax * a.ps_a + bb * a.ps_b + ll * a.ps_l;
            const long long pos = a.pos_bytes == 8 ? __ldg(reinterpret_cast<const long long*>(a.pos) + at) : (long long)__ldg(reinterpret_cast<const int*>(a.pos) + at);
            const unsigned long long turn = __ldg(a.turns + p) * (unsigned long long)pos;
            sincospif((float)(int)(turn >> 32) * 0x1p-31f, &s, &c);
        }
        s_cs[i] = make_float2(c, s);
    }
    __syncthreads();
    // (cos, sin) of the lane's eight pairs; elements that do not turn are left alone (not multiplied by 1 and 0: an infinity would become NaN)
    f32x2 cs[4], sn[4];
    const bool turn0 = INTER ? c0 * 8 < a.R : lane < r16, turn1 = INTER ? c1 * 8 < a.R : turn0;
    {
        const float2* mine = s_cs + (group >> a.lanes_log2) * half;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            float2 u = make_float2(1.f, 0.f), w = u;
            if (m < 2 ? turn0 : turn1) {
                const int p = INTER ? (m < 2 ? c0 * 4 + 2 * m : c1 * 4 + 2 * m - 4) : lane * 8 + 2 * m;
                u = mine[p]; w = mine[p + 1];
            }
            cs[m] = pack2(u.x, w.x); sn[m] = pack2(u.y, w.y);
        }
    }
    const unsigned mask = ((1u << LPR) - 1u) << (threadIdx.x & 31 & ~(LPR - 1));      // the lanes of a row: they go the same way

    auto rows_of = [&](auto role_) {
        constexpr int ROLE = decltype(role_)::value;
        constexpr bool CODES = PAGED && ROLE != ROLE_Q;
        const int row0 = ROLE == ROLE_Q ? 0 : ROLE == ROLE_K ? k_row : v_row, behind = min(end, ROLE == ROLE_Q ? k_row : ROLE == ROLE_K ? v_row : end);
        if (h >= behind) return;
        const int head0 = h - row0;
        // factors: one for a row, or one for every element, the same for all heads (held) or not (loaded with each row)
        const float* w = ROLE == ROLE_Q ? a.qw : ROLE == ROLE_K ? a.kw : nullptr;
        const long long wh = ROLE == ROLE_Q ? a.qw_h : a.kw_h, wd = ROLE == ROLE_Q ? a.qw_d : a.kw_d;
        f32x2 wx[4], wy[4];
        auto load_weights = [&](int head) {
            float g[2][8];
            const float* p = w + head * wh;
            if (ROLE == ROLE_Q ? a.qw_vec : a.kw_vec) {
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < 2; ++j) *reinterpret_cast<float4*>(&g[e][4 * j]) = __ldg(reinterpret_cast<const float4*>(p) + (e ? c1 : c0) * 2 + j);
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[e][j] = __ldg(p + ((e ? c1 : c0) * 8 + j) * wd);
            }
            const Pairs<INTER> z(g);
#pragma unroll
            for (int m = 0; m < 4; ++m) { wx[m] = z.x[m]; wy[m] = z.y[m]; }
        };
        const int weights = !w ? 0 : !wd ? 1 : !wh ? 2 : 3;    // none; one for a row; held; of each head
        if (weights == 2) load_weights(head0);
        // where the rows go
        O* out = nullptr;
        long long out_step = 0;
        size_t at = 0;
        const int bits = ROLE == ROLE_V ? a.c.vb : a.c.kb;
        if constexpr (CODES) {
            const int page_mask = (1 << a.c.page_shift) - 1;
            at = kept ? (((size_t)(slot >> a.c.page_shift) * a.c.H + head0) << a.c.page_shift) + ((uint32_t)slot & page_mask) : 0;
            out_step = (long long)step << a.c.page_shift;
        } else {
            out = ROLE == ROLE_Q ? reinterpret_cast<O*>(a.qo) + b * a.qo_b + l * a.qo_l + head0 * a.qo_h : reinterpret_cast<O*>(a.ko) + b * a.ko_b + l * a.ko_l + head0 * a.ko_h;
            out += c0 * 8;
            out_step = step * (ROLE == ROLE_Q ? a.qo_h : a.ko_h);
        }
        const float most = paged_most(bits), most_inv = paged_most_inv(bits);
#pragma unroll 1
        for (; h < behind; h += step) {
            Piece<T, VEC> f[2];
            if constexpr (RING) {
                asm volatile("cp.async.wait_group %0;" ::"n"(ROT_AHEAD - 2) : "memory");
                const uint4* from = reinterpret_cast<const uint4*>(ring + stage);
                f[0].r.r = from[0];
                f[1].r.r = from[ROT_THREADS<PAGED>];
                stage = stage == (ROT_AHEAD - 1) * STAGE ? 0 : stage + STAGE;
            } else { f[0] = held[0]; f[1] = held[1]; }
            float v[2][8];
            f[0].r.get(v[0]);
            f[1].r.get(v[1]);
            request();
            if constexpr (ROLE != ROLE_V) {
                Pairs<INTER> z(v);
                float factor = 1.f;
                if (a.norm) {
                    auto squares = [&]() -> float {
                        f32x2 s0 = mul2(z.x[0], z.x[0]), s1 = mul2(z.y[0], z.y[0]);
#pragma unroll
                        for (int m = 1; m < 4; ++m) { s0 = fma2(z.x[m], z.x[m], s0); s1 = fma2(z.y[m], z.y[m], s1); }
                        const float2 u = unpack2(s0), y = unpack2(s1);
                        float sum = (u.x + u.y) + (y.x + y.y);
#pragma unroll
                        for (int n = LPR / 2; n; n >>= 1) sum += __shfl_xor_sync(mask, sum, n);
                        return sum;
                    };
                    float sum = squares();
                    // Rows whose norm lies outside of 2^-40 .. 2^40 or below eps (and rows that are no numbers; in all lanes of a row) are divided by it here, in front of their
                    // factors, whose products with the elements alone may be subnormal or infinite.  Squares that leave fp32 (norms from 2^64 on): of the row times 2^-68 they
                    // sum up to 2^127 at most, and eps is nothing next to them.  fp16 has no such rows but zeros.  (Every row divided in front of its factors: registers, and
                    // up to 17 % of the time.  The test costs bf16, first case above, 45.2 -> 45.7 us, last one 83.5 -> 85.2)
                    if (!std::is_same<T, __half>::value && __float_as_uint(sum) - a.fair > a.fair_span) {
                        const bool far = sum == INFINITY;
                        auto scale = [&](float f) {
                            const f32x2 ff = pack2(f, f);
#pragma unroll
                            for (int m = 0; m < 4; ++m) { z.x[m] = mul2(z.x[m], ff); z.y[m] = mul2(z.y[m], ff); }
                        };
                        if (far) { scale(0x1p-68f); sum = squares(); }
                        sum = fmaf(sum, a.sum_mul, far ? 0.f : a.sum_add);
                        scale(sum < a.least && !far ? a.inv_eps : rsqrt_normal(sum));
                    } else {
                        sum = fmaf(sum, a.sum_mul, a.sum_add);
                        factor = std::is_same<T, __half>::value && sum < a.least ? a.inv_eps : rsqrt_normal(sum);      // (fp16: 0 becomes 0 / eps)
                    }
                }
                if (weights == 1) factor *= __ldg(w + (h - row0) * wh);
                else if (weights) {
                    if (weights == 3) load_weights(h - row0);
#pragma unroll
                    for (int m = 0; m < 4; ++m) { z.x[m] = mul2(z.x[m], wx[m]); z.y[m] = mul2(z.y[m], wy[m]); }
                }
                const f32x2 ff = pack2(factor, factor);
#pragma unroll
                for (int m = 0; m < 4; ++m) { z.x[m] = mul2(z.x[m], ff); z.y[m] = mul2(z.y[m], ff); }
                auto turn = [&](int m) {
                    const float2 xc = unpack2(mul2(z.x[m], cs[m])), u = unpack2(z.y[m]), s = unpack2(sn[m]);
                    z.y[m] = fma2(z.y[m], cs[m], mul2(z.x[m], sn[m]));
                    z.x[m] = pack2(fmaf(-u.x, s.x, xc.x), fmaf(-u.y, s.y, xc.y));
                };
                if constexpr (INTER) {
                    if (turn0) { turn(0); turn(1); }
                    if (turn1) { turn(2); turn(3); }
                } else if (turn0) { turn(0); turn(1); turn(2); turn(3); }
                z.values(v);
            }
            if constexpr (CODES) {
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = max_abs(top, v[e][j]);
#pragma unroll
                for (int n = LPR / 2; n; n >>= 1) top = max_abs(top, __shfl_xor_sync(mask, top, n));
                if (kept) {
                    const PagedRow row(top, most, most_inv, a.qeps);
                    int32_t* to = (ROLE == ROLE_V ? a.c.vc : a.c.kc) + at * (D * bits / 32);
                    uint32_t q[2][8];
                    row.codes(v, q);
                    store_codes(to, c0, bits, q[0]);
                    store_codes(to, c1, bits, q[1]);
                    if (lane == 0) (ROLE == ROLE_V ? a.c.vs : a.c.ks)[at] = row.scale;
                }
                at += out_step;
            } else {
                store_piece<O, VEC>(out, v[0]);
                store_piece<O, VEC>(out + apart, v[1]);
                out += out_step;
            }
        }
    };
    rows_of(IsRole<ROLE_Q>());
    rows_of(IsRole<ROLE_K>());
    if constexpr (PAGED) rows_of(IsRole<ROLE_V>());
}

int rotary_args(const char* who, RotArgs& a, const varq_rotary_t* r, int q_heads, int k_heads, int v_heads, int D) {
    if (!r) return fail(VARQ_ERR_ARG, "%s: null rotary descriptor", who);
    if (r->rotary_dim < 16 || r->rotary_dim > D || r->rotary_dim % 16) return fail(VARQ_ERR_UNSUPPORTED, "%s: rotary_dim %d is not a multiple of 16 up to head_dim %d", who, r->rotary_dim, D);
    if (r->n_axes < 1) return fail(VARQ_ERR_ARG, "%s: %d axes", who, r->n_axes);
    if (r->pos_bytes != 4 && r->pos_bytes != 8) return fail(VARQ_ERR_ARG, "%s: positions have 4 or 8 bytes (got %d)", who, r->pos_bytes);
    if (r->norm != VARQ_NORM_NONE && r->norm != VARQ_NORM_L2 && r->norm != VARQ_NORM_RMS) return fail(VARQ_ERR_ARG, "%s: norm %d", who, r->norm);
    if (r->norm != VARQ_NORM_NONE && !(r->eps >= 1e-18f && r->eps < 1e18f)) return fail(VARQ_ERR_ARG, "%s: eps of the norm must lie in [1e-18, 1e18)", who);
    if (q_heads < 0 || k_heads < 0) return fail(VARQ_ERR_ARG, "%s: %d query heads, %d key heads", who, q_heads, k_heads);
    // a lane group's rows are counted in an int, up to four steps (each below 2^17) behind the last one
    if ((long long)q_heads + k_heads + v_heads >= (1ll << 31) - (1 << 20))
        return fail(VARQ_ERR_UNSUPPORTED, "%s: %d query heads, %d key heads: 2^31 - 2^20 rows of a token or more", who, q_heads, k_heads);
    a.turns = reinterpret_cast<const unsigned long long*>(r->turns); a.axis = r->axis; a.pos = r->positions;
    a.pos_bytes = r->pos_bytes; a.n_axes = r->n_axes; a.R = r->rotary_dim; a.inter = r->interleaved != 0;
    a.ps_a = r->pos_stride_axis; a.ps_b = r->pos_stride_b; a.ps_l = r->pos_stride_l;
    a.norm = r->norm;
    a.inv_eps = 1.f / r->eps; a.least = r->norm == VARQ_NORM_L2 ? r->eps * r->eps : -1.f;
    a.sum_mul = r->norm == VARQ_NORM_L2 ? 1.f : 1.f / (float)D; a.sum_add = r->norm == VARQ_NORM_L2 ? 0.f : r->eps;
    const float fair = a.least > 0x1p-80f ? a.least : 0x1p-80f, most = fair > 0x1p80f ? fair : 0x1p80f;
    memcpy(&a.fair, &fair, 4);
    memcpy(&a.fair_span, &most, 4);
    a.fair_span -= a.fair;
    a.half = FastDiv((uint32_t)r->rotary_dim / 2);
    a.qw = r->q_weight; a.qw_h = r->q_weight_stride_h; a.qw_d = r->q_weight_stride_d;
    a.kw = r->k_weight; a.kw_h = r->k_weight_stride_h; a.kw_d = r->k_weight_stride_d;
    a.qw_vec = aligned16(a.qw) && a.qw_d == 1 && a.qw_h % 4 == 0; a.kw_vec = aligned16(a.kw) && a.kw_d == 1 && a.kw_h % 4 == 0;
    return VARQ_OK;
}
int rotary_pointers(const char* who, const RotArgs& a) {
    if (!a.turns || !a.axis || !a.pos) return fail(VARQ_ERR_ARG, "%s: null pointer", who);
    if ((uintptr_t)a.turns % 8 || (uintptr_t)a.axis % 4 || (uintptr_t)a.pos % a.pos_bytes || (uintptr_t)a.qw % 4 || (uintptr_t)a.kw % 4) return fail(VARQ_ERR_ARG, "%s: misaligned pointer", who);
    return VARQ_OK;
}

// Rows of a token side by side: four (neighbours in memory, one warp's worth at 128 columns) where the tokens alone give every SM some warps, more where they are few: a row
// more on a group of lanes spreads its angles and addresses over more rows, a group more keeps more rows in flight.  Threads per SM from which on it is four, us for
// 300 / 1000 tokens of 32 + 4 and of 48 rows: rotate 256: 4.0 / 6.3, 512: 3.9 / 6.5, 1024: 4.1 / 8.2 (1777 tokens 9.3 / 8.1 / 9.3); append 256: 5.8 / 8.7, 512: 8.2 / 10.6.
template <typename T, typename O, int D, bool VEC, bool PAGED> int run_rotary(RotArgs& a, cudaStream_t st) {
    constexpr int LPR = D / 16, GROUPS = ROT_THREADS<PAGED> / LPR;
    const int rows = a.Hq + a.Hk + a.Hv;
    int lanes = 4;
    while (lanes < rows && (unsigned long long)a.tokens * lanes * LPR < (PAGED ? 256ull : 512ull) * sm_count()) lanes *= 2;
    a.lanes_log2 = 0;
    while ((1 << a.lanes_log2) < lanes && (1 << a.lanes_log2) < GROUPS) ++a.lanes_log2;
    a.parts = lanes > GROUPS ? lanes / GROUPS : 1;
    const int tb = GROUPS >> a.lanes_log2;
    const unsigned long long blocks = ((unsigned long long)a.tokens + tb - 1) / tb * a.parts;
    if (blocks > 0x7fffffffull) return fail(VARQ_ERR_UNSUPPORTED, "varq_rotate: more than 2^31 thread blocks");
    const size_t smem = (size_t)tb * (a.R / 2) * sizeof(float2) + (VEC && sizeof(T) == 2 ? ROT_AHEAD * 2 * ROT_THREADS<PAGED> * 16 : 0);
    const auto kernel = a.inter ? rotary_kernel<T, O, D, VEC, PAGED, true> : rotary_kernel<T, O, D, VEC, PAGED, false>;
    VARQ_CUDA_TRY(launch_pdl(kernel, (unsigned)blocks, ROT_THREADS<PAGED>, smem, st, 1, a));
    count_launches(1);
    return VARQ_OK;
}
template <typename T, typename O, bool PAGED> int run_rotary(RotArgs& a, int D, bool vec, cudaStream_t st) {
    return D == 64 ? (vec ? run_rotary<T, O, 64, true, PAGED>(a, st) : run_rotary<T, O, 64, false, PAGED>(a, st))
                   : (vec ? run_rotary<T, O, 128, true, PAGED>(a, st) : run_rotary<T, O, 128, false, PAGED>(a, st));
}
bool rows4_aligned16(const varq_tensor_t* t) {
    const int es = dtype_size(t->dtype);
    return rows_aligned16(t->ptr, t->stride_l, t->stride_h, es) && (t->stride_b * es) % 16 == 0;
}

}  // namespace
}  // namespace varq

using namespace varq;

extern "C" int varq_rotate(const varq_rotary_t* r, const varq_tensor_t* q, const varq_tensor_t* k, int32_t B, int32_t L, int32_t q_heads, int32_t k_heads,
                           int32_t head_dim, const varq_tensor_t* q_out, const varq_tensor_t* k_out, void* stream) {
    RotArgs a = RotArgs();
    if (head_dim != 64 && head_dim != 128) return fail(VARQ_ERR_UNSUPPORTED, "varq_rotate: head_dim %d is not 64 or 128", head_dim);
    if (int rc = rotary_args("varq_rotate", a, r, q_heads, k_heads, 0, head_dim)) return rc;
    if (!q || !k || !q_out || !k_out) return fail(VARQ_ERR_ARG, "varq_rotate: null descriptor");
    if (B < 0 || L < 0) return fail(VARQ_ERR_ARG, "varq_rotate: negative size");
    if (!dtype_ok(q->dtype) || k->dtype != q->dtype) return fail(VARQ_ERR_ARG, "varq_rotate: q and k must have one type, fp32, fp16 or bf16");
    if ((q_out->dtype != q->dtype && q_out->dtype != VARQ_F32) || k_out->dtype != q_out->dtype) return fail(VARQ_ERR_ARG, "varq_rotate: outputs have q's type or fp32, both one");
    const long long n_tokens = (long long)B * L;              // below 2^31, before it is multiplied by heads of up to 2^32
    if (n_tokens >= 0x7fffffffLL || n_tokens * ((long long)q_heads + k_heads) >= 0x7fffffffLL) return fail(VARQ_ERR_UNSUPPORTED, "varq_rotate: 2^31 rows or more");
    if (B == 0 || L == 0 || q_heads + k_heads == 0) return VARQ_OK;
    if (int rc = rotary_pointers("varq_rotate", a)) return rc;
    if ((q_heads && (!q->ptr || !q_out->ptr)) || (k_heads && (!k->ptr || !k_out->ptr))) return fail(VARQ_ERR_ARG, "varq_rotate: null pointer");
    const int es = dtype_size(q->dtype), eo = dtype_size(q_out->dtype);
    if (((uintptr_t)q->ptr | (uintptr_t)k->ptr) % es || ((uintptr_t)q_out->ptr | (uintptr_t)k_out->ptr) % eo) return fail(VARQ_ERR_ARG, "varq_rotate: misaligned pointer");
    a.q = q->ptr; a.qs_b = q->stride_b; a.qs_l = q->stride_l; a.qs_h = q->stride_h;
    a.k = k->ptr; a.ks_b = k->stride_b; a.ks_l = k->stride_l; a.ks_h = k->stride_h;
    a.qo = q_out->ptr; a.qo_b = q_out->stride_b; a.qo_l = q_out->stride_l; a.qo_h = q_out->stride_h;
    a.ko = k_out->ptr; a.ko_b = k_out->stride_b; a.ko_l = k_out->stride_l; a.ko_h = k_out->stride_h;
    a.Hq = q_heads; a.Hk = k_heads; a.Hv = 0;
    a.tokens = (uint32_t)B * (uint32_t)L; a.L = FastDiv((uint32_t)L);
    const bool vec = (!q_heads || (rows4_aligned16(q) && rows4_aligned16(q_out))) && (!k_heads || (rows4_aligned16(k) && rows4_aligned16(k_out)));
    const cudaStream_t st = (cudaStream_t)stream;
    if (q->dtype == VARQ_F32) return run_rotary<float, float, false>(a, head_dim, vec, st);
    if (q->dtype == VARQ_F16) return q_out->dtype == VARQ_F32 ? run_rotary<__half, float, false>(a, head_dim, vec, st) : run_rotary<__half, __half, false>(a, head_dim, vec, st);
    return q_out->dtype == VARQ_F32 ? run_rotary<__nv_bfloat16, float, false>(a, head_dim, vec, st) : run_rotary<__nv_bfloat16, __nv_bfloat16, false>(a, head_dim, vec, st);
}

extern "C" int varq_paged_append_rotated(const varq_paged_t* cache, const varq_rotary_t* r, const varq_tensor_t* q, const varq_tensor_t* k, const varq_tensor_t* v,
                                         const int64_t* slots, int64_t n_tokens, int32_t q_heads, float eps, const varq_tensor_t* q_out, void* stream) {
    RotArgs a = RotArgs();
    if (int rc = paged_check_cache("varq_paged_append_rotated", cache, a.c)) return rc;
    if (int rc = rotary_args("varq_paged_append_rotated", a, r, q_heads, a.c.H, a.c.H, a.c.D)) return rc;
    if (n_tokens < 0) return fail(VARQ_ERR_ARG, "varq_paged_append_rotated: %lld tokens", (long long)n_tokens);
    if (n_tokens >= 0x7fffffffLL || n_tokens * (2ll * a.c.H + q_heads) >= 0x7fffffffLL)
        return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_append_rotated: %lld tokens of %d and 2 x %d heads are 2^31 rows or more", (long long)n_tokens, q_heads, a.c.H);
    if (!q || !k || !v || !q_out) return fail(VARQ_ERR_ARG, "varq_paged_append_rotated: null descriptor");
    if (!dtype_ok(q->dtype) || k->dtype != q->dtype || v->dtype != q->dtype) return fail(VARQ_ERR_ARG, "varq_paged_append_rotated: q, k and v must have one type, fp32, fp16 or bf16");
    if (q_out->dtype != q->dtype) return fail(VARQ_ERR_ARG, "varq_paged_append_rotated: the output has q's type");
    if (!(eps >= 1e-30f && eps < 1e30f)) return fail(VARQ_ERR_ARG, "varq_paged_append_rotated: eps must lie in [1e-30, 1e30)");
    if (n_tokens == 0) return VARQ_OK;
    if (int rc = rotary_pointers("varq_paged_append_rotated", a)) return rc;
    if ((q_heads && (!q->ptr || !q_out->ptr)) || !k->ptr || !v->ptr || !slots) return fail(VARQ_ERR_ARG, "varq_paged_append_rotated: null pointer");
    const int es = dtype_size(q->dtype);
    if (((uintptr_t)q->ptr | (uintptr_t)k->ptr | (uintptr_t)v->ptr | (uintptr_t)q_out->ptr) % es || (uintptr_t)slots % 8) return fail(VARQ_ERR_ARG, "varq_paged_append_rotated: misaligned pointer");
    a.q = q->ptr; a.qs_l = q->stride_l; a.qs_h = q->stride_h;
    a.k = k->ptr; a.ks_l = k->stride_l; a.ks_h = k->stride_h;
    a.v = v->ptr; a.vs_l = v->stride_l; a.vs_h = v->stride_h;
    a.qo = q_out->ptr; a.qo_l = q_out->stride_l; a.qo_h = q_out->stride_h;
    a.Hq = q_heads; a.Hk = a.Hv = a.c.H;
    a.tokens = (uint32_t)n_tokens; a.L = FastDiv((uint32_t)n_tokens);
    a.slots = reinterpret_cast<const long long*>(slots); a.qeps = eps;
    const bool vec = (!q_heads || (rows_aligned16(q->ptr, a.qs_l, a.qs_h, es) && rows_aligned16(q_out->ptr, a.qo_l, a.qo_h, es))) &&
                     rows_aligned16(k->ptr, a.ks_l, a.ks_h, es) && rows_aligned16(v->ptr, a.vs_l, a.vs_h, es);
    const cudaStream_t st = (cudaStream_t)stream;
    return q->dtype == VARQ_F32 ? run_rotary<float, float, true>(a, a.c.D, vec, st) : q->dtype == VARQ_F16 ? run_rotary<__half, __half, true>(a, a.c.D, vec, st)
                                                                                                           : run_rotary<__nv_bfloat16, __nv_bfloat16, true>(a, a.c.D, vec, st);
}
