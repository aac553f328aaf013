// Writing tokens into a paged cache and reading them back.
//
// Append: a row (token, head) of K or V becomes D codes and one scale,
//   scale = max(amax|x| / (2^(bits-1) - 1), eps),   code = rint(x / scale) to even,
// with the bits of a true fp32 division.  Two pieces of eight values per lane, 4 or 8 lanes per row, the row read once and held in registers.  Rounding
// without a division per value: with r = 1 / scale the quotient lies between x r (1 - 2^-21) and x r (1 + 2^-21); each end is rounded by one multiply-add with
// 1.5 * 2^23, which leaves the integer in the low mantissa bits, and where the two agree on all of a lane's values those are the codes.  Else the lane divides.
// The scale's own division by 1, 7 or 127 is Markstein's: with c = RN(1 / d) and q = RN(a c), RN(q + RN(a - q d) c) is RN(a / d), the remainder being exact.
// A row with a NaN or an infinity has a NaN scale and zero codes: whoever reads it gets NaN, as from arithmetic on the values themselves, and whoever does
// not see it loses nothing.
// Read: code * scale, converted to the output's type once.
//
// What bounds them (B200): a read its bytes, 32768 tokens of 8 heads x 128 from 8-bit codes to 16-bit values 37 us = 5.5 TB/s (the copy rate is 6.5).  An append
// of the same size takes 48 us, 31 by its bytes, and fills no unit: issue 66 %, logic pipe 62 %, DRAM 43 %, and waiting for a row's loads is its largest stall.  Both together: 135 us with eight values a lane and a division and its rounding for each, 93 with sixteen
// and the bracket, 85 with Markstein's scale and narrow codes merged by the byte (their bytes alone take 52).  On random values at most one lane in five hundred
// finds its bracket open and divides (16 values, each within 127 * 2^-20 of a tie).  Short calls are a launch's latency: 8 or 999 tokens, written and read
// back, 8.1 us for both launches.
#include "varq_attn.cuh"
#include "varq_codes.cuh"
#include "varq_paged.cuh"
#include "varq_quant.cuh"

namespace varq {
namespace {

struct AppendArgs {
    PagedView c;
    const void *k, *v;
    long long ks_t, ks_h, vs_t, vs_h;
    const long long* slots;
    uint32_t rows;                     // tokens x heads
    FastDiv heads;
    float eps;
};
struct ReadArgs {
    PagedView c;
    void *k, *v;
    long long ks_t, ks_h, vs_t, vs_h;
    const long long* slots;
    uint32_t rows;
    FastDiv heads;
};

constexpr int ROW_THREADS = 256;

// codes of eight values (fp32 with the code in the low mantissa bits) as piece `ch` of a row: 64, 32 or 16 bits
__device__ __forceinline__ void store_codes(int32_t* row, int ch, int bits, const uint32_t (&q)[8]) {
    uint32_t w[2];                     // a byte each
#pragma unroll
    for (int i = 0; i < 2; ++i)
        w[i] = __byte_perm(__byte_perm(q[4 * i], q[4 * i + 1], 0x0040), __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040), 0x5410);
    if (bits == 8) {
        reinterpret_cast<uint2*>(row)[ch] = make_uint2(w[0], w[1]);
    } else if (bits == 4) {            // two in a byte: in bytes 0 and 2
#pragma unroll
        for (int i = 0; i < 2; ++i) { w[i] &= 0x0f0f0f0fu; w[i] |= w[i] >> 4; }
        row[ch] = (int32_t)__byte_perm(w[0], w[1], 0x6420);
    } else {                           // four in a byte: in byte 0
#pragma unroll
        for (int i = 0; i < 2; ++i) { w[i] &= 0x03030303u; w[i] |= w[i] >> 6; w[i] |= w[i] >> 12; }
        reinterpret_cast<unsigned short*>(row)[ch] = (unsigned short)__byte_perm(w[0], w[1], 0x0040);
    }
}
__device__ __forceinline__ void load_codes(const int32_t* row, int ch, int bits, uint32_t (&w)[2]) {
    if (bits == 8) {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(row) + ch);
        w[0] = x.x; w[1] = x.y;
    } else {
        w[0] = bits == 4 ? (uint32_t)__ldg(row + ch) : __ldg(reinterpret_cast<const unsigned short*>(row) + ch);
        w[1] = 0;
    }
}
// signed fields -> fp32: 0x4B000000 | u is 2^23 + u; narrow ones by way of exact fp16 pairs
__device__ __forceinline__ void codes_to_float(const uint32_t (&w)[2], int bits, float (&f)[8]) {
    if (bits == 8) {
        const uint32_t a = w[0] ^ 0x80808080u, b = w[1] ^ 0x80808080u;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(__byte_perm(i < 4 ? a : b, 0x4B000000u, 0x7540 | (i & 3))) - 8388736.f;
    } else if (bits == 4) {                                  // pairs (i, i + 4): 1024 + u, or 1024 + 16 u
        const uint32_t u = w[0] ^ 0x88888888u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t x = i < 2 ? u : u >> 8;
            const uint32_t h = i & 1 ? h2_fma((x & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, 0xD480D480u) : h2_add((x & 0x000F000Fu) | 0x64006400u, 0xE408E408u);
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
            f[i] = v.x; f[i + 4] = v.y;
        }
    } else {
        const uint32_t u = w[0] ^ 0xAAAAu;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(((u >> (2 * i)) & 3u) | 0x4B000000u) - 8388610.f;
    }
}

// eight consecutive values of a row, packed as they come, and their largest absolute value as bits (order of the absolute values, NaN above infinity)
template <typename T, bool VEC> struct Piece {
    Vec8<T> r;
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (VEC) r.load(p);
        else {
            T e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = p[i];
            if constexpr (sizeof(T) == 4) { r.a = make_float4(e[0], e[1], e[2], e[3]); r.b = make_float4(e[4], e[5], e[6], e[7]); }
            else r.r = *reinterpret_cast<const uint4*>(e);
        }
    }
    __device__ __forceinline__ uint32_t top() const {       // 16-bit types: of the even and the odd values, side by side
        if constexpr (sizeof(T) == 4) {
            float v[8];
            r.get(v);
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
            return m;
        } else {
            return __vmaxu2(__vmaxu2(r.r.x & 0x7fff7fffu, r.r.y & 0x7fff7fffu), __vmaxu2(r.r.z & 0x7fff7fffu, r.r.w & 0x7fff7fffu));
        }
    }
};
template <typename T> __device__ __forceinline__ uint32_t merge_top(uint32_t a, uint32_t b) { return sizeof(T) == 4 ? max(a, b) : __vmaxu2(a, b); }
template <typename T> __device__ __forceinline__ float top_value(uint32_t m) {                 // the value itself
    if constexpr (sizeof(T) == 4) return __uint_as_float(m);
    else {
        const unsigned short b = (unsigned short)max(m & 0xffffu, m >> 16);
        return to_f32<T>(*reinterpret_cast<const T*>(&b));
    }
}
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

template <typename T, int D, int U, bool VEC>
__global__ void __launch_bounds__(ROW_THREADS) paged_append_kernel(AppendArgs a) {
    constexpr int LPR = D / 16, RPB = ROW_THREADS / LPR;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & (LPR - 1), page_mask = (1 << a.c.page_shift) - 1;
    const bool is_v = blockIdx.y != 0;
    const T* x = reinterpret_cast<const T*>(is_v ? a.v : a.k);
    const long long st = is_v ? a.vs_t : a.ks_t, sh = is_v ? a.vs_h : a.ks_h;
    const int bits = is_v ? a.c.vb : a.c.kb, words = D * bits / 32;
    int32_t* pool = is_v ? a.c.vc : a.c.kc;
    float* scales = is_v ? a.c.vs : a.c.ks;
    const long long n_slots = (long long)a.c.n_pages << a.c.page_shift;
    const float most = (float)((1 << (bits - 1)) - 1), inv = bits == 8 ? 1.f / 127.f : bits == 4 ? 1.f / 7.f : 1.f;
    const uint32_t row0 = blockIdx.x * (RPB * U) + threadIdx.x / LPR;
    Piece<T, VEC> f[U][2];
    uint32_t at[U];                    // row of the pools
    bool there[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t row = row0 + u * RPB;
        there[u] = false;
        if (row < a.rows) {
            const uint32_t t = a.heads.div(row), h = row - t * a.heads.d;
            const long long slot = __ldg(a.slots + t);
            if ((unsigned long long)slot < (unsigned long long)n_slots) {
                there[u] = true;
                at[u] = (((uint32_t)(slot >> a.c.page_shift) * a.c.H + h) << a.c.page_shift) + ((uint32_t)slot & page_mask);
                const T* p = x + t * st + h * sh + lane * 8;
                f[u][0].load(p);
                f[u][1].load(p + D / 2);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        uint32_t m = there[u] ? merge_top<T>(f[u][0].top(), f[u][1].top()) : 0u;
#pragma unroll
        for (int z = LPR / 2; z; z >>= 1) m = merge_top<T>(m, __shfl_xor_sync(0xffffffffu, m, z));
        if (!there[u]) continue;
        const float top = top_value<T>(m);
        const bool fine = top <= 3.402823466e38f;
        const float quot = top * inv, scale = fine ? fmaxf(fmaf(fmaf(-quot, most, top), inv, quot), a.eps) : __uint_as_float(0x7fffffffu);
        float r;                                             // within 2^-23, as long as it is a normal number
        asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(scale));
        const float lo = r * (1.f - 0x1p-21f), hi = r * (1.f + 0x1p-21f);
        const uint32_t small = scale > 0x1p125f ? 1u : 0u;
        int32_t* out = pool + (size_t)at[u] * words;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float v[8];
            uint32_t q[8], differ = small;
            f[u][e].r.get(v);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float2 x2 = make_float2(v[i], v[i + 1]), magic = make_float2(Q_MAGIC, Q_MAGIC);
                const float2 y = fma_pair(x2, make_float2(lo, lo), magic), z = fma_pair(x2, make_float2(hi, hi), magic);
                q[i] = __float_as_uint(y.x); q[i + 1] = __float_as_uint(y.y);
                differ |= (q[i] ^ __float_as_uint(z.x)) | (q[i + 1] ^ __float_as_uint(z.y));
            }
            if (!fine) {
#pragma unroll
                for (int i = 0; i < 8; ++i) q[i] = 0u;
            } else if (differ) {
#pragma unroll
                for (int i = 0; i < 8; ++i) q[i] = __float_as_uint(rintf(__fdiv_rn(v[i], scale)) + Q_MAGIC);
            }
            store_codes(out, lane + e * LPR, bits, q);
        }
        if (lane == 0) scales[at[u]] = scale;
    }
}

template <typename T, int D, int U, bool VEC>
__global__ void __launch_bounds__(ROW_THREADS) paged_read_kernel(ReadArgs a) {
    constexpr int LPR = D / 16, RPB = ROW_THREADS / LPR;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & (LPR - 1), page_mask = (1 << a.c.page_shift) - 1;
    const bool is_v = blockIdx.y != 0;
    T* out = reinterpret_cast<T*>(is_v ? a.v : a.k);
    const long long st = is_v ? a.vs_t : a.ks_t, sh = is_v ? a.vs_h : a.ks_h;
    const int bits = is_v ? a.c.vb : a.c.kb, words = D * bits / 32;
    const int32_t* pool = is_v ? a.c.vc : a.c.kc;
    const float* scales = is_v ? a.c.vs : a.c.ks;
    const long long n_slots = (long long)a.c.n_pages << a.c.page_shift;
    const uint32_t row0 = blockIdx.x * (RPB * U) + threadIdx.x / LPR;
    uint32_t w[U][2][2];
    T* to[U];
    float s[U];
    bool there[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t row = min(row0 + u * RPB, a.rows - 1), t = a.heads.div(row), h = row - t * a.heads.d;
        const long long slot = __ldg(a.slots + t);
        there[u] = (unsigned long long)slot < (unsigned long long)n_slots;
        to[u] = out + t * st + h * sh + lane * 8;
        w[u][0][0] = w[u][0][1] = w[u][1][0] = w[u][1][1] = 0; s[u] = 0.f;
        if (there[u]) {
            const uint32_t at = (((uint32_t)(slot >> a.c.page_shift) * a.c.H + h) << a.c.page_shift) + ((uint32_t)slot & page_mask);
            const int32_t* p = pool + (size_t)at * words;
            load_codes(p, lane, bits, w[u][0]);
            load_codes(p, lane + LPR, bits, w[u][1]);
            s[u] = __ldg(scales + at);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (row0 + u * RPB >= a.rows) break;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float f[8];
            codes_to_float(w[u][e], bits, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = there[u] ? f[i] * s[u] : 0.f;
            store_vals<T, 8, VEC>(to[u] + e * (D / 2), f, 8);
        }
    }
}

bool rows_aligned16(const void* p, long long st, long long sh, int es) {
    return aligned16(p) && (st * es) % 16 == 0 && (sh * es) % 16 == 0;
}

int check_cache(const char* who, const varq_paged_t* c, PagedView& v) {
    if (!c) return fail(VARQ_ERR_ARG, "%s: null cache", who);
    if (c->n_pages < 1 || c->n_heads < 1) return fail(VARQ_ERR_ARG, "%s: %d pages, %d heads", who, c->n_pages, c->n_heads);
    if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
        return fail(VARQ_ERR_ARG, "%s: a page holds 16, 32, ... 1024 tokens (got %d)", who, c->page_size);
    if (c->head_dim != 64 && c->head_dim != 128) return fail(VARQ_ERR_UNSUPPORTED, "%s: head_dim %d is not 64 or 128", who, c->head_dim);
    if ((c->k_bits != 2 && c->k_bits != 4 && c->k_bits != 8) || (c->v_bits != 2 && c->v_bits != 4 && c->v_bits != 8))
        return fail(VARQ_ERR_ARG, "%s: bits must be 2, 4 or 8 (got %d, %d)", who, c->k_bits, c->v_bits);
    if (!c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale) return fail(VARQ_ERR_ARG, "%s: null pool", who);
    if (!aligned16(c->k_codes) || !aligned16(c->v_codes) || !aligned16(c->k_scale) || !aligned16(c->v_scale)) return fail(VARQ_ERR_ARG, "%s: pools must start on a 16-byte boundary", who);
    if ((unsigned long long)c->n_pages * c->n_heads * c->page_size >= (1ull << 32))
        return fail(VARQ_ERR_UNSUPPORTED, "%s: %d pages of %d tokens and %d heads are 2^32 rows or more", who, c->n_pages, c->page_size, c->n_heads);
    v.kc = c->k_codes; v.vc = c->v_codes; v.ks = c->k_scale; v.vs = c->v_scale;
    v.n_pages = c->n_pages; v.page_shift = 0;
    while ((1 << v.page_shift) < c->page_size) ++v.page_shift;
    v.H = c->n_heads; v.D = c->head_dim; v.kb = c->k_bits; v.vb = c->v_bits;
    return VARQ_OK;
}
int check_rows(const char* who, const PagedView& c, long long n) {
    if (n < 0) return fail(VARQ_ERR_ARG, "%s: %lld tokens", who, n);
    if (n * c.H >= 0x7fffffffLL) return fail(VARQ_ERR_UNSUPPORTED, "%s: %lld tokens of %d heads are 2^31 rows or more", who, n, c.H);
    return VARQ_OK;
}

// Rows per thread: two keep more bytes in flight once the call fills every SM four times over, one spreads a shorter call over the SMs.
// One / two / four rows, 32768 tokens of 8 heads x 128, 8 bits: append of 16-bit values 56.4 / 50.1 / 59.6 us, of fp32 (half the tokens) 32.0 / 33.5 / 48; read
// 41.5 / 37.0 / 42.7 us.
template <int U, typename A, typename K1, typename KU>
int launch_rows(K1 one, KU several, const A& a, int D, cudaStream_t st) {
    const uint32_t rpb = ROW_THREADS / (D / 16);
    if (a.rows >= 4ull * U * rpb * sm_count()) VARQ_CUDA_TRY(launch_pdl(several, dim3((a.rows + U * rpb - 1) / (U * rpb), 2), ROW_THREADS, 0, st, 1, a));
    else VARQ_CUDA_TRY(launch_pdl(one, dim3((a.rows + rpb - 1) / rpb, 2), ROW_THREADS, 0, st, 1, a));
    count_launches(1);
    return VARQ_OK;
}
template <typename T, int D, bool VEC> int run_append(const AppendArgs& a, cudaStream_t st) {
    return launch_rows<2>(paged_append_kernel<T, D, 1, VEC>, paged_append_kernel<T, D, 2, VEC>, a, D, st);
}
template <typename T> int run_append(const AppendArgs& a, bool vec, cudaStream_t st) {
    return a.c.D == 64 ? (vec ? run_append<T, 64, true>(a, st) : run_append<T, 64, false>(a, st)) : (vec ? run_append<T, 128, true>(a, st) : run_append<T, 128, false>(a, st));
}
template <typename T, int D, bool VEC> int run_read(const ReadArgs& a, cudaStream_t st) {
    return launch_rows<2>(paged_read_kernel<T, D, 1, VEC>, paged_read_kernel<T, D, 2, VEC>, a, D, st);
}
template <typename T> int run_read(const ReadArgs& a, bool vec, cudaStream_t st) {
    return a.c.D == 64 ? (vec ? run_read<T, 64, true>(a, st) : run_read<T, 64, false>(a, st)) : (vec ? run_read<T, 128, true>(a, st) : run_read<T, 128, false>(a, st));
}

__device__ int g_paged_status = 0;

}  // namespace

int paged_status_word(int** out) {
    static int* known[64] = {nullptr};                       // per device; the address of a variable of the module does not change
    int dev = 0;
    VARQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && known[dev]) { *out = known[dev]; return VARQ_OK; }
    void* p = nullptr;
    VARQ_CUDA_TRY(cudaGetSymbolAddress(&p, g_paged_status));
    *out = reinterpret_cast<int*>(p);
    if (dev >= 0 && dev < 64) known[dev] = *out;
    return VARQ_OK;
}
int paged_status(int* out) {
    if (int rc = paged_attn_tc_status(out)) return rc;
    int v = 0;
    VARQ_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_paged_status, sizeof(int)));
    if (v != 0) {
        const int zero = 0;
        VARQ_CUDA_TRY(cudaMemcpyToSymbol(g_paged_status, &zero, sizeof(int)));
    }
    if (*out == 0) *out = v;
    return VARQ_OK;
}

}  // namespace varq

using namespace varq;

extern "C" int varq_paged_append(const varq_paged_t* cache, const varq_tensor_t* k, const varq_tensor_t* v, const int64_t* slots, int64_t n_tokens,
                                 float eps, void* stream) {
    AppendArgs a;
    if (int rc = check_cache("varq_paged_append", cache, a.c)) return rc;
    if (int rc = check_rows("varq_paged_append", a.c, n_tokens)) return rc;
    if (!k || !v) return fail(VARQ_ERR_ARG, "varq_paged_append: null descriptor");
    if (!dtype_ok(k->dtype) || k->dtype != v->dtype) return fail(VARQ_ERR_ARG, "varq_paged_append: K and V must have one type, fp32, fp16 or bf16");
    if (!(eps >= 1e-30f && eps < 1e30f)) return fail(VARQ_ERR_ARG, "varq_paged_append: eps must lie in [1e-30, 1e30)");
    if (n_tokens == 0) return VARQ_OK;
    if (!k->ptr || !v->ptr || !slots) return fail(VARQ_ERR_ARG, "varq_paged_append: null pointer");
    const int es = dtype_size(k->dtype);
    if ((uintptr_t)k->ptr % es || (uintptr_t)v->ptr % es || (uintptr_t)slots % 8) return fail(VARQ_ERR_ARG, "varq_paged_append: misaligned pointer");
    a.k = k->ptr; a.v = v->ptr;
    a.ks_t = k->stride_l; a.ks_h = k->stride_h; a.vs_t = v->stride_l; a.vs_h = v->stride_h;
    a.slots = reinterpret_cast<const long long*>(slots);
    a.rows = (uint32_t)(n_tokens * a.c.H);
    a.heads = FastDiv((uint32_t)a.c.H);
    a.eps = eps;
    const bool vec = rows_aligned16(k->ptr, a.ks_t, a.ks_h, es) && rows_aligned16(v->ptr, a.vs_t, a.vs_h, es);
    const cudaStream_t st = (cudaStream_t)stream;
    return k->dtype == VARQ_F32 ? run_append<float>(a, vec, st) : k->dtype == VARQ_F16 ? run_append<__half>(a, vec, st) : run_append<__nv_bfloat16>(a, vec, st);
}

extern "C" int varq_paged_read(const varq_paged_t* cache, const int64_t* slots, int64_t n_tokens, const varq_tensor_t* k_out,
                               const varq_tensor_t* v_out, void* stream) {
    ReadArgs a;
    if (int rc = check_cache("varq_paged_read", cache, a.c)) return rc;
    if (int rc = check_rows("varq_paged_read", a.c, n_tokens)) return rc;
    if (!k_out || !v_out) return fail(VARQ_ERR_ARG, "varq_paged_read: null descriptor");
    if (!dtype_ok(k_out->dtype) || k_out->dtype != v_out->dtype) return fail(VARQ_ERR_ARG, "varq_paged_read: K and V must have one type, fp32, fp16 or bf16");
    if (n_tokens == 0) return VARQ_OK;
    if (!k_out->ptr || !v_out->ptr || !slots) return fail(VARQ_ERR_ARG, "varq_paged_read: null pointer");
    const int es = dtype_size(k_out->dtype);
    if ((uintptr_t)k_out->ptr % es || (uintptr_t)v_out->ptr % es || (uintptr_t)slots % 8) return fail(VARQ_ERR_ARG, "varq_paged_read: misaligned pointer");
    a.k = k_out->ptr; a.v = v_out->ptr;
    a.ks_t = k_out->stride_l; a.ks_h = k_out->stride_h; a.vs_t = v_out->stride_l; a.vs_h = v_out->stride_h;
    a.slots = reinterpret_cast<const long long*>(slots);
    a.rows = (uint32_t)(n_tokens * a.c.H);
    a.heads = FastDiv((uint32_t)a.c.H);
    const bool vec = rows_aligned16(a.k, a.ks_t, a.ks_h, es) && rows_aligned16(a.v, a.vs_t, a.vs_h, es);
    const cudaStream_t st = (cudaStream_t)stream;
    return k_out->dtype == VARQ_F32 ? run_read<float>(a, vec, st) : k_out->dtype == VARQ_F16 ? run_read<__half>(a, vec, st) : run_read<__nv_bfloat16>(a, vec, st);
}

namespace {

// How a call is shared out.
//
// Kernel: few query rows per head of the cache leave most of the chunk kernel's 256 idle, while the decode kernel reads the keys once for every 16.  They cross
// where the decode kernel needs a third row tile at head_dim 128, and a sixth at 64 (chunk kernel / decode kernel of 16 rows a CTA, us):
//   128: 24 rows, 64 sequences of 8000 keys 542 / 391; 32 rows, 8 of 1000 24.1 / 20.4; 40 rows, 64 of 8000 542 / 560; 64 rows, 8 of 1000 24.4 / 30.1
//    64: 40 rows, 32 of 2000 136 / 102; 64 rows 141 / 132; 100 rows, 4 of 300 13.8 / 13.4 (which a larger call would turn round)
// Rows of a decode CTA: 17 to 24 rows in one CTA unpack the keys once, in two of 16 twice, but side by side.  Two / one, us: 24 rows, 64 sequences of 8000 keys, 8 heads
// 391 / 303; 20 rows, 24 sequences, a window of 1024 32.0 / 28.9; 24 rows, 8 sequences of 1000 20.4 / 19.1; with fewer sequences and heads than a quarter of the SMs 24
// rows, 1 sequence of 1000 11.6 / 14.4; 20 rows, 2 of 3000 18.1 / 18.8; at 64 columns, 2 of 4000, 2 bits 15.2 / 15.4.  Two of 24 for 40 rows at 64 columns, instead of three
// of 16: 115 and 102.
// Parts of the key range: more of them fill the SMs, and each costs a CTA its set-up and, through the workspace, a store and a second launch.  The model below
// (in tiles; fixed and merge are fits) picked the best or within 2 % of the best of 1 .. 24 parts on 10 of 11 calls that were measured, e.g. 256 queries
// behind 8192 keys, 8 heads: 1 / 2 / 4 / 8 parts 186 / 117 / 72 / 88 us, picks 4; 2048 behind 16384 740 / 807 / 807 / 943, picks 1.  The one it misses are
// chunks of 17 to 512 queries behind 0 to 4000 keys, 1 / 2 parts 91 / 77 us, picks 1: only the longest length is known here, and there it is the critical path.
// Of 11 calls of the decode kernel it misses one by 10 % (24 sequences, 15 rows, a window of 1024: 25.1 us in clusters of two, 22.8 in two parts through the
// workspace); one query behind 32768 keys takes 313 us in one part, 84 in 4, 31 in 16, 21 in the 54 that it picks.
// Cluster or workspace: parts of the decode kernel that are resident all at once, up to eight of a row tile, meet in a cluster; without a second launch one
// sequence of 1000 keys takes 8.0 us, with it 12.9.  Where they are not resident, clusters wait for room together: 64 sequences of 8000 keys, 16 heads 284 us
// in clusters, 259 through the workspace.
struct AttnPlan {
    bool tc, cluster;                  // kernel; its parts meet in clusters, not in the workspace
    int rows;                          // query rows of a CTA (decode kernel)
    int splits, tiles_per_split;       // tiles of 16 keys (decode kernel)
};
AttnPlan plan_attn(const varq_paged_t* c, const varq_paged_batch_t* b) {
    AttnPlan p;
    const int max_q = (int)(b->max_q < b->n_queries ? b->max_q : b->n_queries), D = c->head_dim;
    const long long rows = (long long)max_q * (b->q_heads / c->n_heads);
    const long long seen = (long long)b->window + max_q + b->sinks, span = b->window && seen < b->max_kv ? seen : b->max_kv;      // keys of a CTA, about
    p.tc = forced_attn_path() == VARQ_ATTN_PATH_TC || (forced_attn_path() != VARQ_ATTN_PATH_DECODE && rows > (D == 64 ? 80 : 32));
    p.rows = rows <= 8 ? 8 : rows > 16 && rows <= 24 && 4ll * b->n_seqs * c->n_heads >= sm_count() ? 24 : 16;
    const long long unit = p.tc ? 128 : 16, tiles = span > unit ? (span + unit - 1) / unit : 1;
    const int resident = p.tc ? 1 : p.rows > 16 ? (D == 128 ? 2 : 3) : p.rows > 8 ? (D == 128 ? 3 : 4) : D == 64 ? 5 : c->k_bits == 8 && c->v_bits == 8 ? 3 : 4;       // CTAs per SM
    const long long base = (long long)b->n_seqs * c->n_heads * (p.tc ? (rows + 255) / 256 : (rows + p.rows - 1) / p.rows), room = (long long)sm_count() * resident;
    // the number of parts that makes the waves of CTAs shortest, a CTA costing its tiles and a fixed part, parts in the workspace those, the second launch, too
    const long long fixed = p.tc ? 4 : 16, least = p.tc ? 2 : 4, merge = p.tc ? 4 : 24;
    long long best = 0;
    p.splits = 1; p.cluster = false;
    for (long long s = 1; s == 1 || (s <= tiles / least && s <= 256); ++s) {
        const bool near = !p.tc && s <= PAGED_CLUSTER && base * s <= room;
        const long long cost = (base * s + room - 1) / room * ((tiles + s - 1) / s + fixed + (s > 1 && p.tc ? fixed : 0)) + (s > 1 && !near ? merge : 0);
        if (best == 0 || cost < best) { best = cost; p.splits = (int)s; p.cluster = s > 1 && near; }
        if (base * s > 8 * room) break;
    }
    p.tiles_per_split = (int)((tiles + p.splits - 1) / p.splits);
    return p;
}
size_t part_floats(const AttnPlan& p, const varq_paged_t* c, const varq_paged_batch_t* b) {
    return p.splits > 1 && !p.cluster ? (size_t)p.splits * b->n_queries * b->q_heads * (c->head_dim + 2) : 0;
}

}  // namespace

extern "C" size_t varq_paged_attn_workspace_bytes(const varq_paged_t* cache, const varq_paged_batch_t* batch) {
    if (!cache || !batch || cache->n_heads < 1 || batch->q_heads < cache->n_heads || batch->n_seqs < 1 || batch->n_queries < 1 || batch->max_q < 1 || batch->max_kv < 0 ||
        batch->window < 0 || batch->sinks < 0 || cache->head_dim < 1)
        return 0;
    return part_floats(plan_attn(cache, batch), cache, batch) * sizeof(float);
}

extern "C" int varq_paged_attn(const varq_paged_t* cache, const varq_paged_batch_t* batch, const varq_tensor_t* q, const varq_tensor_t* out, float* lse,
                               void* workspace, size_t workspace_bytes, void* stream) {
    PagedAttnArgs a;
    if (int rc = check_cache("varq_paged_attn", cache, a.c)) return rc;
    if (!batch || !q || !out) return fail(VARQ_ERR_ARG, "varq_paged_attn: null descriptor");
    if (batch->n_seqs < 0 || batch->n_queries < 0 || batch->max_q < 0 || batch->max_kv < 0 || batch->table_pages < 0)
        return fail(VARQ_ERR_ARG, "varq_paged_attn: negative size");
    if (batch->q_heads < 1 || batch->q_heads % a.c.H) return fail(VARQ_ERR_ARG, "varq_paged_attn: %d query heads over %d heads of the cache", batch->q_heads, a.c.H);
    if ((q->dtype != VARQ_F16 && q->dtype != VARQ_BF16) || out->dtype != q->dtype)
        return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_attn: queries and outputs are fp16 or bf16, both of one type");
    if (batch->window < 0 || batch->sinks < 0) return fail(VARQ_ERR_ARG, "varq_paged_attn: window %d, sinks %d", batch->window, batch->sinks);
    if (batch->window && !batch->causal) return fail(VARQ_ERR_ARG, "varq_paged_attn: a window needs causal attention");
    if (batch->sinks && !batch->window) return fail(VARQ_ERR_ARG, "varq_paged_attn: sinks need a window");
    if (!(batch->softmax_scale > 0.f && batch->softmax_scale < 1e30f)) return fail(VARQ_ERR_ARG, "varq_paged_attn: softmax_scale must be positive and finite");
    if (batch->n_seqs > 65535) return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_attn: %d sequences (65535 at most)", batch->n_seqs);
    if (batch->n_queries >= (1ll << 31)) return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_attn: 2^31 query tokens or more");
    if ((batch->max_q < batch->n_queries ? batch->max_q : batch->n_queries) * (batch->q_heads / a.c.H) >= 0x7fffffffLL - 511)
        return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_attn: %d queries of a sequence, %d query heads over %d: 2^31 - 512 query rows of a head or more", batch->max_q, batch->q_heads, a.c.H);
    if (batch->n_queries == 0 || batch->n_seqs == 0 || batch->max_q == 0) return VARQ_OK;
    if (!q->ptr || !out->ptr || !batch->q_starts || !batch->kv_lens || (batch->table_pages && !batch->block_table)) return fail(VARQ_ERR_ARG, "varq_paged_attn: null pointer");
    if (((uintptr_t)q->ptr | (uintptr_t)out->ptr) % 2 || ((uintptr_t)batch->q_starts | (uintptr_t)batch->kv_lens | (uintptr_t)batch->block_table | (uintptr_t)lse) % 4)
        return fail(VARQ_ERR_ARG, "varq_paged_attn: misaligned pointer");
    a.q = q->ptr; a.dtype = q->dtype; a.qs_t = q->stride_l; a.qs_h = q->stride_h;
    a.out = out->ptr; a.os_t = out->stride_l; a.os_h = out->stride_h;
    a.lse = lse;
    a.q_starts = batch->q_starts; a.kv_lens = batch->kv_lens; a.table = batch->block_table;
    a.table_stride = batch->table_stride; a.table_pages = batch->table_pages;
    a.B = batch->n_seqs; a.T = (int)batch->n_queries; a.Hq = batch->q_heads; a.G = a.Hq / a.c.H;
    a.max_q = (int)(batch->max_q < batch->n_queries ? batch->max_q : batch->n_queries); a.max_kv = batch->max_kv;
    a.scale_log2 = batch->softmax_scale * 1.4426950408889634f;
    a.causal = batch->causal != 0; a.window = batch->window;
    a.sinks = batch->sinks < PAGED_MOST_KEYS ? batch->sinks : PAGED_MOST_KEYS;      // more tokens than there are: all of them
    const AttnPlan p = plan_attn(cache, batch);
    const size_t need = part_floats(p, cache, batch) * sizeof(float);
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(VARQ_ERR_WORKSPACE, "varq_paged_attn: workspace of %zu bytes (16-byte aligned) needed, %zu given", need, workspace_bytes);
    float *ws_o = reinterpret_cast<float*>(workspace), *ws_ml = ws_o + (size_t)p.splits * a.T * a.Hq * a.c.D;
    const cudaStream_t st = (cudaStream_t)stream;
    int* status = nullptr;
    if (int rc = paged_status_word(&status)) return rc;      // the kernels write to it: no launch without it
    if (int rc = p.tc ? paged_attn_tc_run(a, p.splits, ws_o, ws_ml, status, st) : paged_attn_decode_run(a, p.rows, p.splits, p.cluster, p.tiles_per_split, ws_o, ws_ml, status, st)) return rc;
    return need ? paged_attn_merge_run(a, p.splits, ws_o, ws_ml, st) : VARQ_OK;
}
