// Device side of the pool's storage: where a row lies in its block of 16 positions, types of rows, and the signed transform of a row
// that is spread over lanes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "k2t_device.cuh"
#include "k2t_kv_pool.h"

namespace k2t {

// A block holds 16 rows of keys, 16 rows of values, then their scales ([row] fp32, or [row][group of 64] bf16).  8-bit codes are stored
// with their sign bit flipped, 4-bit ones as centroid indices, element 2 i in the low half of byte i.
template <int HD, int BITS> struct PoolBlock {
    static constexpr uint32_t RB = BITS == 8 ? HD : HD / 2, G = BITS == 8 ? 1 : HD / 64, SC = BITS == 8 ? 64 : HD / 2;
    static constexpr uint32_t V_AT = POOL_ROWS * RB, KS_AT = 2 * POOL_ROWS * RB, VS_AT = KS_AT + SC, BYTES = KS_AT + 2 * SC;
};

// Byte `at` of row p (0 .. 15) within 16 rows of RB bytes.  The attention kernel's lanes (n, t) = (lane / 4, lane % 4) read rows 4 (n / 2)
// + n % 2 (and two further) at pieces t of keys, and rows 4 t + i at piece n of values; the order of rows and the exclusive-or of the
// 16-byte pieces put the lanes of one shared-memory phase on different banks in both patterns, for each length of a row.
template <uint32_t RB> __host__ __device__ __forceinline__ constexpr uint32_t row_place(uint32_t p, uint32_t at) {
    static_assert(RB == 128 || RB == 64 || RB == 32, "row of 32, 64 or 128 bytes");
    const uint32_t quad = (p >> 2) & 3u;
    if (RB == 128) return p * 128 + (at ^ (((quad << 1) ^ ((p & 1u) << 2)) << 4));
    if (RB == 64) return (p ^ (quad & 1u)) * 64 + (at ^ ((2u * ((quad ^ (quad >> 1)) & 1u)) << 4));
    return (p ^ ((quad >> 1) | ((quad & 1u) << 1))) * 32 + at;
}

constexpr uint32_t TYPE_F32 = KRONOS_CUDA_TYPE_F32, TYPE_BF16 = KRONOS_CUDA_TYPE_BF16, TYPE_F16 = KRONOS_CUDA_TYPE_F16;

__device__ __forceinline__ float2 unpack2(uint32_t type, uint32_t w) {
    return type == TYPE_BF16 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)) : __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
__device__ __forceinline__ uint32_t pack2(uint32_t type, float x, float y) {
    if (type == TYPE_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// Eight consecutive elements from / to element `at` of rows.  Asking and converting are apart, so that several rows can be on their way: a
// conversion inside the branches on the type would wait for each.
struct Row8 {
    uint32_t w[8];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void ask(const RowsArg &a, size_t at) {
        const uint8_t *p = static_cast<const uint8_t *>(a.p) + at * (a.type == TYPE_F32 ? 4 : 2);
        if (a.wide) {
            const uint4 x = __ldcg(reinterpret_cast<const uint4 *>(p));
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
            if (a.type == TYPE_F32) {
                const uint4 y = __ldcg(reinterpret_cast<const uint4 *>(p) + 1);
                w[4] = y.x; w[5] = y.y; w[6] = y.z; w[7] = y.w;
            }
        } else if (a.type == TYPE_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __ldcg(reinterpret_cast<const uint32_t *>(p) + i);
        } else {
            const uint16_t *q = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldcg(q + 2 * i) | ((uint32_t)__ldcg(q + 2 * i + 1) << 16);
        }
    }
    __device__ __forceinline__ void values(uint32_t type, float (&v)[8]) const {
        if (type == TYPE_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2(type, w[i]);
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
};
__device__ __forceinline__ void rows_put8(const RowsArg &a, size_t at, const float (&v)[8]) {
    if (a.type == TYPE_F32) {
        float *p = static_cast<float *>(a.p) + at;
        if (a.wide) {
            reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = v[i];
        }
        return;
    }
    uint16_t *p = static_cast<uint16_t *>(a.p) + at;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack2(a.type, v[2 * i], v[2 * i + 1]);
    if (a.wide) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) { p[2 * i] = (uint16_t)w[i]; p[2 * i + 1] = (uint16_t)(w[i] >> 16); }
    }
}

// Butterflies over the N elements that a thread holds (distances h0, 2 h0, ..), the lower element a + b, the upper a - b.
template <int N> __device__ __forceinline__ void butterflies_in(float (&v)[N]) {
#pragma unroll
    for (int h = 1; h < N; h *= 2)
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((i & h) == 0) {
                const float a = v[i], b = v[i + h];
                v[i] = __fadd_rn(a, b);
                v[i + h] = __fsub_rn(a, b);
            }
}
// The same between lanes l and l ^ m, all N elements: the other's value plus or minus one's own, rounded once.
template <int N> __device__ __forceinline__ void butterflies_across(float (&v)[N], uint32_t m, uint32_t lane) {
    const float sign = (lane & m) != 0 ? -1.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __fmaf_rn(v[i], sign, __shfl_xor_sync(0xffffffffu, v[i], m));
}
__device__ __forceinline__ float flip(float x, uint32_t signs, int i) { return __uint_as_float(__float_as_uint(x) ^ (signs << (31 - i) & 0x80000000u)); }         // by bit i

// The signs of eight elements times 1/8: one product instead of a shift, an exclusive-or and a product, for kernels that transform several rows.
struct Eighths {
    float f[8];
    __device__ __forceinline__ explicit Eighths(uint32_t signs) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = flip(0.125f, signs, i);
    }
};
// Eight lanes hold 64 values, eight each; (1/8) H64 D x, butterflies in the order 1, 2, .. 32.
__device__ __forceinline__ void transform8(float (&v)[8], const Eighths &e, uint32_t lane) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], e.f[i]);
    butterflies_in(v);
#pragma unroll
    for (uint32_t m = 1; m < 8; m <<= 1) butterflies_across(v, m, lane);
}
__device__ __forceinline__ void transform8_back(float (&v)[8], const Eighths &e, uint32_t lane) {
    butterflies_in(v);
#pragma unroll
    for (uint32_t m = 1; m < 8; m <<= 1) butterflies_across(v, m, lane);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], e.f[i]);
}
__device__ __forceinline__ void transform8(float (&v)[8], uint32_t signs, uint32_t lane) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(flip(v[i], signs, i), 0.125f);
    butterflies_in(v);
#pragma unroll
    for (uint32_t m = 1; m < 8; m <<= 1) butterflies_across(v, m, lane);
}
__device__ __forceinline__ void transform8_back(float (&v)[8], uint32_t signs, uint32_t lane) {
    butterflies_in(v);
#pragma unroll
    for (uint32_t m = 1; m < 8; m <<= 1) butterflies_across(v, m, lane);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = flip(__fmul_rn(v[i], 0.125f), signs, i);
}
__device__ __forceinline__ uint32_t signs8(const PoolView &p, uint32_t at) { return p.signs[at >> 5] >> (at & 31u) & 0xFFu; }

__device__ __forceinline__ uint32_t half2_bits(float x, float y) { const __half2 h = __floats2half2_rn(x, y); return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ uint32_t hsub2(uint32_t x, uint32_t y) {
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&x), *reinterpret_cast<const __half2 *>(&y));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float log2_approx(float x) { float y; asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float rcp_approx(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// The power of two that brings a row's largest value to 2^13 .. 2^14, within what a float and its inverse hold.
__device__ __forceinline__ int query_exponent(float top) { return min(126, max(-126, 140 - (int)((__float_as_uint(top) >> 23) & 255u))); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Eight elements of a query row as operands, the row over HD / 8 lanes: transformed, times a power of two that brings its largest to 2^13 .. 2^14 (so
// that both terms are ordinary halves), and split.  Returns the power's inverse.  Rows that are not there are zeros.
template <int HD> __device__ __forceinline__ float query_halves(const PoolView &pool, const RowsArg &q, bool there, size_t at, uint32_t l, uint32_t lane, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    float v[8], top = 0.0f;
    Row8 x;
    x.clear();
    if (there) x.ask(q, at + l * 8);
    x.values(q.type, v);
    transform8(v, signs8(pool, l * 8), lane);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
    for (uint32_t m = HD / 16; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    const int e = query_exponent(top);
    const float up = power_of_two(e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float y = v[2 * i] * up, z = v[2 * i + 1] * up;
        hi[i] = half2_bits(y, z);
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi[i]));
        lo[i] = half2_bits(y - f.x, z - f.y);
    }
    return power_of_two(-e);
}

// The scale of a value row in the exponents of its weights.  A row of zeros, which has the scale 0, takes one below all that count, so that the
// running maximum is that of the rows an output is made of, however much of the weight the zeros have.  Exponentials reach down to 2^-126, so a
// zero row counts beside values of scales up to 2^62; 4-bit rows with scales below 2^-64 have those as factors of it.  NaN stays NaN.
constexpr float LEAST_SCALE = 0x1p-64f;
__device__ __forceinline__ float weight_scale(float scale) { return scale < LEAST_SCALE ? LEAST_SCALE : scale; }

// A running maximum m stands 7 below the largest exponent that it was set by and follows where one has come 15 above it, so that weights are up to 2^15
// (halves reach 2^16) and those down to 2^-21 of the largest are ordinary halves: the grid of 2^-24 below is 2^-31 of it or finer.
constexpr float MAX_BELOW = 7.0f, MAX_ROOM = 15.0f;

// Constants of the expansion, kept in registers: left to the compiler they are loaded again for every use where registers are short.
struct Expand {
    uint32_t exponent, hi0, hi1, lo0, lo1;
    __device__ __forceinline__ Expand() {
        asm volatile("mov.b32 %0, 0x64646464;" : "=r"(exponent));
        asm volatile("mov.b32 %0, 0x2C1F1206;" : "=r"(hi0));
        asm volatile("mov.b32 %0, 0x7F604B3A;" : "=r"(hi1));
        asm volatile("mov.b32 %0, 0x3A4B607F;" : "=r"(lo0));
        asm volatile("mov.b32 %0, 0x06121F2C;" : "=r"(lo1));
    }
    // Bytes 128 + c (the lower or upper two) as halves c: 0x6400 + byte is 1024 + byte.
    __device__ __forceinline__ uint32_t halves_lo(uint32_t x) const { return hsub2(prmt(x, exponent, 0x4140u), 0x64806480u); }
    __device__ __forceinline__ uint32_t halves_hi(uint32_t x) const { return hsub2(prmt(x, exponent, 0x4342u), 0x64806480u); }
    // Four 4-bit codes (the low 16 bits of w) as bytes 128 + centroid.  A selector with bit 3 set yields a byte's sign, here 0: of the two
    // tables each index finds its magnitude in one and 0 in the other.
    __device__ __forceinline__ uint32_t centroids4(uint32_t w) const { return 0x80808080u + prmt(hi0, hi1, w ^ 0x8888u) - prmt(lo0, lo1, w); }
};

constexpr uint32_t POOL_ERR_PAGE = 6;        // a page or slot outside the pool
__device__ __forceinline__ void pool_bad_page(const PoolView &v) { atomicExch(v.err, POOL_ERR_PAGE); }

}  // namespace k2t
