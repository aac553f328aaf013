// A row (token, head) of K or V on its way into a paged cache, by D / 16 neighbouring lanes with two pieces of eight values each: loads, the largest absolute
// value, scale and codes.  varq_paged.cu says what is done and why.
#pragma once
#include "varq_paged.cuh"
#include "varq_quant.cuh"

namespace varq {

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

__device__ __forceinline__ float paged_most(int bits) { return (float)((1 << (bits - 1)) - 1); }
__device__ __forceinline__ float paged_most_inv(int bits) { return bits == 8 ? 1.f / 127.f : bits == 4 ? 1.f / 7.f : 1.f; }

// scale of a row whose largest absolute value is `top`, and codes of its values
struct PagedRow {
    float scale, lo, hi;
    uint32_t small;
    bool fine;
    __device__ __forceinline__ PagedRow(float top, float most, float inv, float eps) {
        fine = top <= 3.402823466e38f;
        const float quot = top * inv;
        scale = fine ? fmaxf(fmaf(fmaf(-quot, most, top), inv, quot), eps) : __uint_as_float(0x7fffffffu);
        float r;                                             // within 2^-23, as long as it is a normal number
        asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(scale));
        lo = r * (1.f - 0x1p-21f); hi = r * (1.f + 0x1p-21f);
        small = scale > 0x1p125f ? 1u : 0u;
    }
    // the codes of a piece or two, in the low mantissa bits of `q`
    __device__ __forceinline__ void codes(const float (&v)[8], uint32_t (&q)[8]) const {
        fix(v, q, bracket(v, q));
    }
    __device__ __forceinline__ void codes(const float (&v)[2][8], uint32_t (&q)[2][8]) const {
        const uint32_t differ = bracket(v[0], q[0]) | bracket(v[1], q[1]);
        if (!fine || differ) { fix(v[0], q[0], differ); fix(v[1], q[1], differ); }
    }
private:
    // one end of the bracket; nonzero where the other end may be another integer
    __device__ __forceinline__ uint32_t bracket(const float (&v)[8], uint32_t (&q)[8]) const {
        uint32_t differ = small;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 x2 = make_float2(v[i], v[i + 1]), magic = make_float2(Q_MAGIC, Q_MAGIC);
            const float2 y = fma_pair(x2, make_float2(lo, lo), magic), z = fma_pair(x2, make_float2(hi, hi), magic);
            q[i] = __float_as_uint(y.x); q[i + 1] = __float_as_uint(y.y);
            differ |= (q[i] ^ __float_as_uint(z.x)) | (q[i + 1] ^ __float_as_uint(z.y));
        }
        return differ;
    }
    __device__ __forceinline__ void fix(const float (&v)[8], uint32_t (&q)[8], uint32_t differ) const {
        if (!fine) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = 0u;
        } else if (differ) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = __float_as_uint(rintf(__fdiv_rn(v[i], scale)) + Q_MAGIC);
        }
    }
};

// 16-byte accesses of every row
inline bool rows_aligned16(const void* p, long long st, long long sh, int es) { return aligned16(p) && (st * es) % 16 == 0 && (sh * es) % 16 == 0; }

}  // namespace varq
