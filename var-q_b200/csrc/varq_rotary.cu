// Norms of queries and keys per head and the rotation by position, in one pass: on their own (varq_rotate), and in front of a paged cache, where the
// rotated keys are quantized straight into their slots (varq_paged_append_rotated).
//
//   x <- x / max(|x|_2, eps)  or  x / sqrt(mean x^2 + eps)  or  x;   x <- x w;   (a, b) <- (a cos t - b sin t, b cos t + a sin t)
//
// for pairs (a, b) of neighbours or of elements half the rotary dimension apart, t = position on the pair's axis times its frequency.
// Angles: a frequency is held as turns per position, a fraction of 64 bits; position times that, modulo 2^64, is the angle in turns with an error of
// position * 2^-65 turns (a product in fp32 is off by whole radians from 10^7 on).  Its upper 32 bits go to sincospi.  Everything
// behind is fp32, rounded once to the output's type, or to the code of the cache.
//
// D / 16 neighbouring lanes hold a row with two pieces of eight values each, chosen so that both values of a pair are in one lane.  The lanes of a
// token share its angles, which the block computes once for all heads.
#include "varq_paged_rows.cuh"

namespace varq {
namespace {

constexpr int ROT_THREADS = 256;

struct RotArgs {
    const unsigned long long* turns; const int32_t* axis; const void* pos;
    int pos_bytes, n_axes, R, inter;
    long long ps_a, ps_b, ps_l;
    int norm; float eps;
    const float *qw, *kw; long long qw_h, qw_d, kw_h, kw_d;
    const void *q, *k, *v; long long qs_b, qs_l, qs_h, ks_b, ks_l, ks_h, vs_l, vs_h;
    void *qo, *ko; long long qo_b, qo_l, qo_h, ko_b, ko_l, ko_h;
    int Hq, Hk, Hv;
    uint32_t tokens; FastDiv L;
    int lanes_log2, parts;            // rows of a token that a block works on side by side (log2), parts of a token's rows
    PagedView c; const long long* slots; float qeps;
};

template <typename T, typename O, int D, bool VEC, bool PAGED, int U>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(RotArgs a) {
    constexpr int LPR = D / 16, GROUPS = ROT_THREADS / LPR;
    extern __shared__ float2 s_cs[];                         // [token][pair]: cos, sin
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & (LPR - 1), group = threadIdx.x / LPR, side = 1 << a.lanes_log2;
    const int tb = GROUPS >> a.lanes_log2, half = a.R >> 1;
    const uint32_t block = blockIdx.x / (uint32_t)a.parts, part = blockIdx.x - block * (uint32_t)a.parts;
    const uint32_t t0 = block * tb, t = t0 + (uint32_t)(group >> a.lanes_log2);
    const bool token_there = t < a.tokens;
    const uint32_t b = token_there ? a.L.div(t) : 0, l = token_there ? t - b * a.L.d : 0;
    const int rows = a.Hq + a.Hk + a.Hv, first = (int)part * side + (group & (side - 1)), step = side * a.parts;
    // pieces of a lane: 8 values each, from c0 * 8 and c1 * 8 on
    const int r16 = a.R >> 4;
    const int c0 = a.inter ? lane : lane < r16 ? lane : 2 * lane, c1 = a.inter ? lane + LPR : lane < r16 ? lane + r16 : 2 * lane + 1;
    long long slot = -1;
    if (PAGED && token_there) slot = __ldg(a.slots + t);
    const bool kept = PAGED && (unsigned long long)slot < ((unsigned long long)a.c.n_pages << a.c.page_shift);

    Piece<T, VEC> f[U][2];
    auto fetch = [&](int h, Piece<T, VEC> (&p)[2]) {
        if (!token_there || h >= rows) return;
        const T* x;
        if (h < a.Hq) x = reinterpret_cast<const T*>(a.q) + b * a.qs_b + l * a.qs_l + h * a.qs_h;
        else if (h < a.Hq + a.Hk) x = reinterpret_cast<const T*>(a.k) + b * a.ks_b + l * a.ks_l + (h - a.Hq) * a.ks_h;
        else x = reinterpret_cast<const T*>(a.v) + l * a.vs_l + (h - a.Hq - a.Hk) * a.vs_h;
        p[0].load(x + c0 * 8);
        p[1].load(x + c1 * 8);
    };
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(first + u * step, f[u]);

    // ---- angles of the block's tokens
    for (int i = threadIdx.x; i < tb * half; i += ROT_THREADS) {
        const int tk = i / half, p = i - tk * half;
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
    // (cos, sin) of the lane's eight pairs
    float cs[8], sn[8];
    const float2* mine = s_cs + (group >> a.lanes_log2) * half;
    const bool turn0 = a.inter ? c0 * 8 < a.R : lane < r16, turn1 = a.inter ? c1 * 8 < a.R : false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float2 x = make_float2(1.f, 0.f);
        if (a.inter) { if (i < 4 ? turn0 : turn1) x = mine[(i < 4 ? c0 * 4 : c1 * 4 - 4) + i]; }
        else if (turn0) x = mine[lane * 8 + i];
        cs[i] = x.x; sn[i] = x.y;
    }
    const int page_mask = (1 << a.c.page_shift) - 1;

    auto work = [&](int h, const Piece<T, VEC> (&p)[2]) {
        const bool there = token_there && h < rows, is_q = h < a.Hq, is_k = !is_q && h < a.Hq + a.Hk;
        float v[2][8];
        p[0].r.get(v[0]);
        p[1].r.get(v[1]);
        const float* w = is_q ? a.qw : a.kw;
        const long long wh = is_q ? a.qw_h : a.kw_h, wd = is_q ? a.qw_d : a.kw_d;
        const int head = is_q ? h : is_k ? h - a.Hq : h - a.Hq - a.Hk;
        float factor = 1.f;
        if (a.norm) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum = fmaf(v[e][i], v[e][i], sum);
#pragma unroll
            for (int z = LPR / 2; z; z >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, z);
            if (a.norm == VARQ_NORM_L2) {
                const float length = sqrtf(sum);
                factor = 1.f / (length < a.eps ? a.eps : length);      // (a NaN stays one)
            } else factor = 1.f / sqrtf(sum * (1.f / D) + a.eps);
        }
        if (is_q || is_k) {
            if (w && there) {
                if (wd == 0) {
                    const float m = __ldg(w + head * wh);
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[e][i] = v[e][i] * factor * m;
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[e][i] = v[e][i] * factor * __ldg(w + head * wh + ((e ? c1 : c0) * 8 + i) * wd);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[e][i] *= factor;
            }
            if (a.inter) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (!(e ? turn1 : turn0)) continue;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = v[e][2 * i], y = v[e][2 * i + 1], c = cs[4 * e + i], s = sn[4 * e + i];
                        v[e][2 * i] = fmaf(x, c, -(y * s));
                        v[e][2 * i + 1] = fmaf(y, c, x * s);
                    }
                }
            } else if (turn0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = v[0][i], y = v[1][i], c = cs[i], s = sn[i];
                    v[0][i] = fmaf(x, c, -(y * s));
                    v[1][i] = fmaf(y, c, x * s);
                }
            }
        }
        if (PAGED) {
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[e][i]) & 0x7fffffffu);
#pragma unroll
            for (int z = LPR / 2; z; z >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, z));
            if (!is_q) {
                if (!there || !kept) return;
                const int bits = is_k ? a.c.kb : a.c.vb;
                const uint32_t at = (((uint32_t)(slot >> a.c.page_shift) * a.c.H + head) << a.c.page_shift) + ((uint32_t)slot & page_mask);
                const PagedRow row(__uint_as_float(m), paged_most(bits), paged_most_inv(bits), a.qeps);
                int32_t* out = (is_k ? a.c.kc : a.c.vc) + (size_t)at * (D * bits / 32);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t q[8];
                    row.codes(v[e], q);
                    store_codes(out, e ? c1 : c0, bits, q);
                }
                if (lane == 0) (is_k ? a.c.ks : a.c.vs)[at] = row.scale;
                return;
            }
        }
        if (!there) return;
        O* o = is_q ? reinterpret_cast<O*>(a.qo) + b * a.qo_b + l * a.qo_l + head * a.qo_h : reinterpret_cast<O*>(a.ko) + b * a.ko_b + l * a.ko_l + head * a.ko_h;
        store_vals<O, 8, VEC>(o + c0 * 8, v[0], 8);
        store_vals<O, 8, VEC>(o + c1 * 8, v[1], 8);
    };
    // every warp takes every turn: lanes without a row keep its shuffles company
    for (int i = (int)part * side; i < rows; i += U * step) {
        const int h = first + (i - (int)part * side);
        Piece<T, VEC> g[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) fetch(h + (U + u) * step, g[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) work(h + u * step, f[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) { f[u][0] = g[u][0]; f[u][1] = g[u][1]; }
    }
}

int rotary_args(const char* who, RotArgs& a, const varq_rotary_t* r, int q_heads, int k_heads, int D) {
    if (!r) return fail(VARQ_ERR_ARG, "%s: null rotary descriptor", who);
    if (r->rotary_dim < 16 || r->rotary_dim > D || r->rotary_dim % 16) return fail(VARQ_ERR_UNSUPPORTED, "%s: rotary_dim %d is not a multiple of 16 up to head_dim %d", who, r->rotary_dim, D);
    if (r->n_axes < 1) return fail(VARQ_ERR_ARG, "%s: %d axes", who, r->n_axes);
    if (r->pos_bytes != 4 && r->pos_bytes != 8) return fail(VARQ_ERR_ARG, "%s: positions have 4 or 8 bytes (got %d)", who, r->pos_bytes);
    if (r->norm != VARQ_NORM_NONE && r->norm != VARQ_NORM_L2 && r->norm != VARQ_NORM_RMS) return fail(VARQ_ERR_ARG, "%s: norm %d", who, r->norm);
    if (r->norm != VARQ_NORM_NONE && !(r->eps >= 1e-30f && r->eps < 1e30f)) return fail(VARQ_ERR_ARG, "%s: eps of the norm must lie in [1e-30, 1e30)", who);
    if (q_heads < 0 || k_heads < 0) return fail(VARQ_ERR_ARG, "%s: %d query heads, %d key heads", who, q_heads, k_heads);
    a.turns = reinterpret_cast<const unsigned long long*>(r->turns); a.axis = r->axis; a.pos = r->positions;
    a.pos_bytes = r->pos_bytes; a.n_axes = r->n_axes; a.R = r->rotary_dim; a.inter = r->interleaved != 0;
    a.ps_a = r->pos_stride_axis; a.ps_b = r->pos_stride_b; a.ps_l = r->pos_stride_l;
    a.norm = r->norm; a.eps = r->eps;
    a.qw = r->q_weight; a.qw_h = r->q_weight_stride_h; a.qw_d = r->q_weight_stride_d;
    a.kw = r->k_weight; a.kw_h = r->k_weight_stride_h; a.kw_d = r->k_weight_stride_d;
    return VARQ_OK;
}
int rotary_pointers(const char* who, const RotArgs& a) {
    if (!a.turns || !a.axis || !a.pos) return fail(VARQ_ERR_ARG, "%s: null pointer", who);
    if ((uintptr_t)a.turns % 8 || (uintptr_t)a.axis % 4 || (uintptr_t)a.pos % a.pos_bytes || (uintptr_t)a.qw % 4 || (uintptr_t)a.kw % 4) return fail(VARQ_ERR_ARG, "%s: misaligned pointer", who);
    return VARQ_OK;
}

// Rows of a token side by side: four (neighbours in memory, one warp's worth at 128 columns) where the tokens alone fill the chip, more where they are few.
template <typename T, typename O, int D, bool VEC, bool PAGED> int run_rotary(RotArgs& a, cudaStream_t st) {
    constexpr int LPR = D / 16, GROUPS = ROT_THREADS / LPR;
    const int rows = a.Hq + a.Hk + a.Hv;
    int lanes = 4;
    while (lanes < rows && (unsigned long long)a.tokens * lanes * LPR < 1024ull * sm_count()) lanes *= 2;
    a.lanes_log2 = 0;
    while ((1 << a.lanes_log2) < lanes && (1 << a.lanes_log2) < GROUPS) ++a.lanes_log2;
    a.parts = lanes > GROUPS ? lanes / GROUPS : 1;
    const int tb = GROUPS >> a.lanes_log2;
    const unsigned long long blocks = ((unsigned long long)a.tokens + tb - 1) / tb * a.parts;
    if (blocks > 0x7fffffffull) return fail(VARQ_ERR_UNSUPPORTED, "varq_rotate: more than 2^31 thread blocks");
    VARQ_CUDA_TRY(launch_pdl(rotary_kernel<T, O, D, VEC, PAGED, 2>, (unsigned)blocks, ROT_THREADS, (size_t)tb * (a.R / 2) * sizeof(float2), st, 1, a));
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
    RotArgs a{};
    if (head_dim != 64 && head_dim != 128) return fail(VARQ_ERR_UNSUPPORTED, "varq_rotate: head_dim %d is not 64 or 128", head_dim);
    if (int rc = rotary_args("varq_rotate", a, r, q_heads, k_heads, head_dim)) return rc;
    if (!q || !k || !q_out || !k_out) return fail(VARQ_ERR_ARG, "varq_rotate: null descriptor");
    if (B < 0 || L < 0) return fail(VARQ_ERR_ARG, "varq_rotate: negative size");
    if (!dtype_ok(q->dtype) || k->dtype != q->dtype) return fail(VARQ_ERR_ARG, "varq_rotate: q and k must have one type, fp32, fp16 or bf16");
    if ((q_out->dtype != q->dtype && q_out->dtype != VARQ_F32) || k_out->dtype != q_out->dtype) return fail(VARQ_ERR_ARG, "varq_rotate: outputs have q's type or fp32, both one");
    if ((long long)B * L * ((long long)q_heads + k_heads) >= 0x7fffffffLL) return fail(VARQ_ERR_UNSUPPORTED, "varq_rotate: 2^31 rows or more");
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
    RotArgs a{};
    if (int rc = paged_check_cache("varq_paged_append_rotated", cache, a.c)) return rc;
    if (int rc = rotary_args("varq_paged_append_rotated", a, r, q_heads, a.c.H, a.c.D)) return rc;
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
