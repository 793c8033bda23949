// Rows of the pool: written (signed transform, quantisation, block keys of full pages), read back, and the choice of pages by block keys.
// The arithmetic of a row is that of the engines' caches (store_hadamard_q8_head*_raw, store_hadamard_q4_head_raw, nf4_nearest_idx,
// src/model/real_llm.rs:8303-8365, 8615-8701), operation by operation in fp32, so codes and scales are the same bits.
#include <algorithm>

#include "k2t_kv_pool.cuh"

namespace k2t {
namespace {

// The nearest of the 16 centroids.  The magnitude is a sum of steps at the borders between magnitudes: a comparison that yields 1.0 or 0.0 and a
// fused multiply-add each, on two pipes, where a tree of selections keeps one busy twice as long.
__device__ __forceinline__ float at_least(float a, float border) { float s; asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(s) : "f"(a), "f"(border)); return s; }
__device__ __forceinline__ float with_sign(float x, float of) { return __uint_as_float(__float_as_uint(x) | (__float_as_uint(of) & 0x80000000u)); }          // x >= 0
__device__ __forceinline__ float nearest_value(float y) {
    const float a = fabsf(y);
    float c = __fmaf_rn(at_least(a, 12.0f), 12.0f, 6.0f);
    c = __fmaf_rn(at_least(a, 24.5f), 13.0f, c);
    c = __fmaf_rn(at_least(a, 37.5f), 13.0f, c);
    c = __fmaf_rn(at_least(a, 51.0f), 14.0f, c);
    c = __fmaf_rn(at_least(a, 66.5f), 17.0f, c);
    c = __fmaf_rn(at_least(a, 85.5f), 21.0f, c);
    c = __fmaf_rn(at_least(a, 111.5f), 31.0f, c);
    return with_sign(c, __fadd_rn(y, 0.0f));          // + 0 takes the sign of -0
}
__device__ __forceinline__ float nearest_index(float y) {          // 0 .. 15
    const float a = fabsf(y);
    const float low = __fadd_rn(__fadd_rn(at_least(a, 12.0f), at_least(a, 24.5f)), at_least(a, 37.5f)), high = __fadd_rn(__fadd_rn(at_least(a, 51.0f), at_least(a, 66.5f)), __fadd_rn(at_least(a, 85.5f), at_least(a, 111.5f)));
    return __fadd_rn(7.5f, with_sign(__fadd_rn(__fadd_rn(low, 0.5f), high), __fadd_rn(y, 0.0f)));
}
constexpr float SMALLEST = 1.1920929e-07f;       // 8-bit rows up to here are stored as zeros
// Rounded to the nearest whole number, the even one of two: the low byte of the result.  |x| <= 2^22.
__device__ __forceinline__ uint32_t rounded_byte(float x) { return __float_as_uint(__fadd_rn(x, 12582912.0f)); }
__device__ __forceinline__ uint32_t four_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return prmt(prmt(a, b, 0x0040u), prmt(c, d, 0x0040u), 0x5410u); }
// Byte i of w, which holds 128 + c, as c: 0x4B0000xx is 2^23 + xx.
__device__ __forceinline__ float signed_byte(uint32_t w, uint32_t i) { return __fsub_rn(__uint_as_float(prmt(w, 0x4B000000u, 0x7540u + i)), 8388736.0f); }

// The largest magnitude of a row over LANES lanes, as bits: these are ordered as the magnitudes are, with infinities and NaN above all others.
constexpr uint32_t INFINITE = 0x7F800000u;
template <int LANES, int N> __device__ __forceinline__ uint32_t top_bits(const float (&v)[N]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
    return top;
}
// A row over LANES lanes, eight values each, as 8-bit codes: what all quantised rows of 8 bits share.  `scale` is NaN for a row that is
// not finite (its codes are 0).
template <int LANES, int N> __device__ __forceinline__ void quantise8(const float (&v)[N], uint32_t (&code)[N], float &scale) {          // codes: the low bytes
    const uint32_t bits = top_bits<LANES>(v);
    const float top = __uint_as_float(bits);
    const bool bad = bits >= INFINITE, zero = bad || top <= SMALLEST;
    const float inv = zero ? 0.0f : __fdiv_rn(127.0f, top);
#pragma unroll
    for (int i = 0; i < N; ++i) code[i] = rounded_byte(bad ? 0.0f : __fmul_rn(v[i], inv));
    scale = bad ? __uint_as_float(0x7FC00000u) : zero ? 0.0f : __fdiv_rn(top, 127.0f);
}

// Where (slot, head) lies: the block and the row in it; null for a slot that is left out.
__device__ __forceinline__ uint8_t *block_of(const PoolView &p, int64_t slot, uint32_t head, uint32_t block_bytes, uint32_t &row) {
    if (slot < 0) return nullptr;
    const uint64_t page = (uint64_t)slot >> p.d.page_shift;
    if (page >= p.d.num_pages) { pool_bad_page(p); return nullptr; }
    const uint32_t in = (uint32_t)slot & ((1u << p.d.page_shift) - 1u);
    row = in & (POOL_ROWS - 1);
    return p.rows + (((page * p.d.kv_heads + head) << (p.d.page_shift - 4)) + (in >> 4)) * block_bytes;
}

// ------------------------------------------------------------------------------------------------ rows in, rows out
// head_dim / 8 lanes hold a row, eight values each; rows are numbered (token, keys | values, head).  A thread has its part of ROW_AHEAD rows on
// the way at a time: two (16384 tokens x 8 heads of 128 written and read: one 98, two 95.6, four 96.9 us; 4001 x 32 of 64, 4 bits: 65, 63, 67), or one
// where the rows are too few for the second to hide behind the first.  In us, one | two, by CTAs of one: written, 8 bits, 300 CTAs 2.4 | 2.9, 1200 4.8 | 5.2,
// 2400 8.0 | 8.2, 5000 14.7 | 14.4; 4 bits 300 3.9 | 4.8, 1200 8.8 | 9.6, 5000 29.5 | 28.7; read, 300 2.1 | 2.5, 600 3.3 | 3.0, 2400 6.8 | 6.6.
constexpr uint32_t ROW_THREADS = 256;
struct RowAt { uint32_t t, value, head; };
__device__ __forceinline__ RowAt row_at(const PoolStoreArgs &a, uint32_t r) {          // r below 2^31: a division by a multiplication (and a shift) that is exact there
    const uint32_t per = 2 * a.pool.d.kv_heads, t = __umulhi(r, a.rows_mul) >> a.rows_shift, u = r - t * per, value = u >= a.pool.d.kv_heads ? 1u : 0u;
    return RowAt{t, value, u - value * a.pool.d.kv_heads};
}

// One row, transformed, into its place.
template <int HD, int BITS> __device__ __forceinline__ void put_row(const PoolStoreArgs &a, uint8_t *block, uint32_t row, uint32_t value, uint32_t l, uint32_t lane, float (&v)[8]) {
    using B = PoolBlock<HD, BITS>;
    constexpr uint32_t LANES = HD / 8;
    if (BITS == 8) {
        uint32_t c[8];
        float scale;
        quantise8<LANES>(v, c, scale);
        if (block == nullptr) return;
        *reinterpret_cast<uint2 *>(block + value * B::V_AT + row_place<B::RB>(row, l * 8)) =
            make_uint2(four_bytes(c[0], c[1], c[2], c[3]) ^ 0x80808080u, four_bytes(c[4], c[5], c[6], c[7]) ^ 0x80808080u);
        if (l == 0) reinterpret_cast<float *>(block + (value ? B::VS_AT : B::KS_AT))[row] = scale;
    } else {
        const uint32_t bits = top_bits<8>(v), row_bits = LANES == 8 ? bits : max(bits, __shfl_xor_sync(0xffffffffu, bits, 8));
        const float top = __uint_as_float(bits);
        const bool bad = row_bits >= INFINITE;            // of the whole row: its groups stand or fall together
        const bool zero = top < 1e-30f || bad;
        const float inv0 = zero ? 0.0f : __fdiv_rn(127.0f, top);
        float rc[8], den = 0.0f, num = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = nearest_value(__fmul_rn(v[i], inv0));
            rc[i] = __fmul_rn(v[i], c);
            den = __fmaf_rn(c, c, den);                    // whole numbers below 2^24: in any order
        }
#pragma unroll
        for (int m = 4; m > 0; m >>= 1) den += __shfl_xor_sync(0xffffffffu, den, m);
        // the products are added up in the order of the elements: lane after lane
#pragma unroll
        for (uint32_t s = 0; s < 8; ++s) {
            float n = num;
#pragma unroll
            for (int i = 0; i < 8; ++i) n = __fadd_rn(n, rc[i]);
            num = __shfl_sync(0xffffffffu, n, (lane & ~7u) | s);
        }
        const float fit = den > 1e-12f && num > 0.0f ? __fdiv_rn(num, den) : __fdiv_rn(top, 127.0f);
        const __nv_bfloat16 sb = __float2bfloat16_rn(zero ? 0.0f : fit);
        const float s = __bfloat162float(sb), inv = s > 1e-30f ? __fdiv_rn(1.0f, s) : 0.0f;
        uint32_t half[2];                      // four indices each as one whole number below 2^16
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float n = nearest_index(__fmul_rn(v[4 * i + 3], inv));
#pragma unroll
            for (int j = 2; j >= 0; --j) n = __fmaf_rn(n, 16.0f, nearest_index(__fmul_rn(v[4 * i + j], inv)));
            half[i] = __float_as_uint(__fadd_rn(n, 8388608.0f));
        }
        const uint32_t w = zero ? 0x88888888u : prmt(half[0], half[1], 0x5410u);
        if (block == nullptr) return;
        *reinterpret_cast<uint32_t *>(block + value * B::V_AT + row_place<B::RB>(row, l * 4)) = w;
        if (l % 8 == 0) reinterpret_cast<uint16_t *>(block + (value ? B::VS_AT : B::KS_AT))[row * B::G + l / 8] = bad ? 0x7FC0u : __bfloat16_as_ushort(sb);
    }
}

template <int HD, int BITS, uint32_t ROW_AHEAD> __global__ void __launch_bounds__(ROW_THREADS) pool_store_kernel(const __grid_constant__ PoolStoreArgs a) {
    using B = PoolBlock<HD, BITS>;
    constexpr uint32_t LANES = HD / 8, STEP = ROW_THREADS / LANES;
    const uint32_t lane = threadIdx.x & 31, l = lane % LANES, rows = a.n_tok * 2 * a.pool.d.kv_heads;
    const Eighths signs(signs8(a.pool, l * 8));
    const uint32_t r0 = blockIdx.x * (STEP * ROW_AHEAD) + threadIdx.x / LANES;
    pdl_wait();
    pdl_trigger();
    int64_t slot[ROW_AHEAD];
    Row8 got[ROW_AHEAD];
    RowAt at[ROW_AHEAD];
#pragma unroll
    for (uint32_t u = 0; u < ROW_AHEAD; ++u) {
        const uint32_t r = r0 + u * STEP;
        at[u] = row_at(a, min(r, rows - 1));
        slot[u] = r < rows ? __ldcg(a.slots + at[u].t) : -1;
        const RowsArg &src = at[u].value ? a.v : a.k;
        got[u].ask(src, at[u].t * src.token_stride + at[u].head * src.head_stride + l * 8);
    }
#pragma unroll
    for (uint32_t u = 0; u < ROW_AHEAD; ++u) {
        if (r0 - threadIdx.x / LANES + u * STEP >= rows) break;          // all of the CTA
        uint32_t row = 0;
        uint8_t *block = block_of(a.pool, slot[u], at[u].head, B::BYTES, row);
        float v[8];
        got[u].values(a.k.type, v);
        transform8(v, signs, lane);
        put_row<HD, BITS>(a, block, row, at[u].value, l, lane, v);
    }
}

// N stored values of a row, element N l on, times their scale; l over HD / N lanes.
template <int HD, int BITS, int N> struct Stored {
    using B = PoolBlock<HD, BITS>;
    static constexpr uint32_t BYTES = N * BITS / 8;
    uint32_t w[BYTES > 4 ? 2 : 1], s;
    __device__ __forceinline__ void get(const uint8_t *block, uint32_t rows_at, uint32_t scales_at, uint32_t row, uint32_t l) {
        const uint8_t *p = block + rows_at + row_place<B::RB>(row, l * BYTES);
        if constexpr (BYTES == 8) { const uint2 x = __ldcg(reinterpret_cast<const uint2 *>(p)); w[0] = x.x; w[1] = x.y; }
        else if constexpr (BYTES == 4) w[0] = __ldcg(reinterpret_cast<const uint32_t *>(p));
        else if constexpr (BYTES == 2) w[0] = __ldcg(reinterpret_cast<const uint16_t *>(p));
        else w[0] = __ldcg(p);
        if (BITS == 8) s = __ldcg(reinterpret_cast<const uint32_t *>(block + scales_at) + row);
        else s = (uint32_t)__ldcg(reinterpret_cast<const uint16_t *>(block + scales_at) + row * B::G + l * N / 64) << 16;
    }
    __device__ __forceinline__ void values(const Expand &ex, float (&v)[N]) const {
        const float scale = __uint_as_float(s);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __fmul_rn(signed_byte(BITS == 8 ? w[i / 4] : ex.centroids4(w[0] >> (i / 4 * 16)), i % 4), scale);
    }
};

template <int HD, int BITS, uint32_t ROW_AHEAD> __global__ void __launch_bounds__(ROW_THREADS) pool_load_kernel(const __grid_constant__ PoolStoreArgs a) {
    using B = PoolBlock<HD, BITS>;
    constexpr uint32_t LANES = HD / 8, STEP = ROW_THREADS / LANES;
    const uint32_t lane = threadIdx.x & 31, l = lane % LANES, rows = a.n_tok * 2 * a.pool.d.kv_heads;
    const Eighths signs(signs8(a.pool, l * 8));
    const uint32_t r0 = blockIdx.x * (STEP * ROW_AHEAD) + threadIdx.x / LANES;
    const Expand ex;
    pdl_wait();
    pdl_trigger();
    RowAt at[ROW_AHEAD];
    int64_t slot[ROW_AHEAD];
    Stored<HD, BITS, 8> got[ROW_AHEAD];
    bool live[ROW_AHEAD];
#pragma unroll
    for (uint32_t u = 0; u < ROW_AHEAD; ++u) {
        const uint32_t r = r0 + u * STEP;
        at[u] = row_at(a, min(r, rows - 1));
        slot[u] = r < rows ? __ldcg(a.slots + at[u].t) : -1;
    }
#pragma unroll
    for (uint32_t u = 0; u < ROW_AHEAD; ++u) {
        uint32_t row = 0;
        const uint8_t *block = block_of(a.pool, slot[u], at[u].head, B::BYTES, row);
        live[u] = block != nullptr;
        got[u].get(live[u] ? block : a.pool.rows, at[u].value ? B::V_AT : 0, at[u].value ? B::VS_AT : B::KS_AT, row, l);
    }
#pragma unroll
    for (uint32_t u = 0; u < ROW_AHEAD; ++u) {
        if (r0 - threadIdx.x / LANES + u * STEP >= rows) break;          // all of the CTA
        float v[8];
        got[u].values(ex, v);
        transform8_back(v, signs, lane);
        const RowsArg &dst = at[u].value ? a.v : a.k;
        if (live[u]) rows_put8(dst, at[u].t * dst.token_stride + at[u].head * dst.head_stride + l * 8, v);
    }
}

// ------------------------------------------------------------------------------------------------ block keys
// The mean of a page's keys as they are stored (transformed), summed in the order of their positions, quantised as an 8-bit row.  The
// token that writes a page's last row makes it.  A warp looks over 32 tokens of a head.
template <int HD, int BITS> __global__ void __launch_bounds__(ROW_THREADS) pool_block_key_kernel(const __grid_constant__ PoolStoreArgs a) {
    using B = PoolBlock<HD, BITS>;
    constexpr int N = HD / 32, AHEAD = 16;
    const uint32_t lane = threadIdx.x & 31, kh = a.pool.d.kv_heads, pt = 1u << a.pool.d.page_shift;
    const uint64_t w = (uint64_t)blockIdx.x * (ROW_THREADS / 32) + (threadIdx.x >> 5);
    const uint32_t head = (uint32_t)(w % kh);
    const uint64_t t = w / kh * 32 + lane;
    const Expand ex;
    pdl_wait();
    pdl_trigger();
    const int64_t slot = t < a.n_tok ? __ldcg(a.slots + t) : -1;
    const bool last = slot >= 0 && ((uint32_t)slot & (pt - 1)) == pt - 1 && (uint64_t)slot >> a.pool.d.page_shift < a.pool.d.num_pages;
    for (uint32_t todo = __ballot_sync(0xffffffffu, last); todo != 0; todo &= todo - 1) {
        const uint64_t page = (uint64_t)__shfl_sync(0xffffffffu, slot, __ffs(todo) - 1) >> a.pool.d.page_shift;
        const uint8_t *block = a.pool.rows + ((page * kh + head) << (a.pool.d.page_shift - 4)) * B::BYTES;
        float sum[N];
#pragma unroll
        for (int k = 0; k < N; ++k) sum[k] = 0.0f;
        for (uint32_t i = 0; i < pt; i += AHEAD, block += B::BYTES) {
            Stored<HD, BITS, N> got[AHEAD];
#pragma unroll
            for (uint32_t j = 0; j < AHEAD; ++j) got[j].get(block, 0, B::KS_AT, j, lane);
#pragma unroll
            for (uint32_t j = 0; j < AHEAD; ++j) {
                float v[N];
                got[j].values(ex, v);
#pragma unroll
                for (int k = 0; k < N; ++k) sum[k] = __fadd_rn(sum[k], v[k]);
            }
        }
        const float part = 1.0f / (float)pt;             // a power of two
#pragma unroll
        for (int k = 0; k < N; ++k) sum[k] = __fmul_rn(sum[k], part);
        uint32_t c[N];
        float scale;
        quantise8<32>(sum, c, scale);
        int8_t *to = a.pool.block_keys + (page * kh + head) * HD + lane * N;
        if constexpr (N == 4) *reinterpret_cast<uint32_t *>(to) = four_bytes(c[0], c[1], c[2], c[3]);
        else *reinterpret_cast<uint16_t *>(to) = (uint16_t)prmt(c[0], c[1], 0x0040u);
        if (lane == 0) a.pool.block_key_scales[page * kh + head] = scale;
    }
}

// ------------------------------------------------------------------------------------------------ choice of pages
// CTA = (token, kv head).  The query is the sum of the head's queries, quantised as an 8-bit row; a page scores the whole-number product
// with its block key times the key's scale (one rounding, so that scores are the same wherever they are computed).  The order of
// scores is that of their bits as numbers; the pages are those at or above a threshold (found byte by byte), of its equals the first.
// Two sizes of CTA: with few (token, kv head) pairs the time is one CTA's chain of loads, and 512 threads have a whole sequence's keys in
// flight; with many, smaller CTAs have fewer threads idle at their barriers.  In us, 512 | 128 threads, for tables of 250 / 625 / 2000 pages: 192 pairs
// 8.1 | 10.4, 12.4 | 17.8, 22.5 | 46.7; 400 pairs 12.6 | 11.1, 21 | 18.7, 36.7 | 48.6; 800 pairs 18.9 | 13.7, 32 | 23, 59.6 | 61.3; 2000 pairs 40 | 23, 70 | 41, 133 | 111.
__device__ __forceinline__ uint32_t ordered(float x) {           // NaN behind everything
    if (x != x) return 0;
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <int HD, uint32_t SEL_THREADS> __global__ void __launch_bounds__(SEL_THREADS, 2048 / SEL_THREADS / 2) pool_select_kernel(const __grid_constant__ PoolAttnArgs a) {
    constexpr uint32_t SEL_WARPS = SEL_THREADS / 32;
    extern __shared__ uint32_t s_key[];
    __shared__ __align__(16) int8_t s_q[HD];
    __shared__ uint32_t s_warp[2][SEL_WARPS], s_hist[256], s_pick[3];
    __shared__ float s_rows[SEL_WARPS][HD], s_sum[HD];
    const PoolShape &d = a.pool.d;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, t = blockIdx.x / d.kv_heads, h = blockIdx.x % d.kv_heads, group = a.heads / d.kv_heads;
    pdl_wait();
    pdl_trigger();
    const int32_t seen = __ldcg(a.lens + t), seq = a.seq != nullptr ? __ldcg(a.seq + t) : (int32_t)t;
    const uint32_t len = seq < 0 ? 0u : (uint32_t)max(0, seen);
    uint32_t n = (uint32_t)(((uint64_t)len + (1u << d.page_shift) - 1) >> d.page_shift);
    if (n > a.pages_stride) {
        n = a.pages_stride;
        if (tid == 0) pool_bad_page(a.pool);
    }
    int32_t *out = a.chosen + ((size_t)t * d.kv_heads + h) * a.top;
    if (n <= a.top) {                     // every page
        for (uint32_t i = tid; i < a.top; i += SEL_THREADS) out[i] = i < n ? (int32_t)i : -1;
        return;
    }
    // eight lanes read a block key, four pages at a time; the first ones are on their way while the query is made
    constexpr uint32_t W = HD / 32, AHEAD = 4;              // words of a lane
    const int32_t *table = a.pages + (size_t)seq * a.pages_stride;
    const uint32_t from = a.sinks, to = n - a.local, sub = lane & 7u;          // of these pages the best: n > top >= sinks + local
    uint32_t key[AHEAD][W];
    float scale[AHEAD];
    auto ask = [&](uint32_t i0) {
        int32_t page[AHEAD];
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u) {
            const uint32_t i = i0 + u * SEL_WARPS * 4 + lane / 8;
            page[u] = i < to ? __ldcg(table + i) : 0;
        }
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u) {
            const bool bad = page[u] < 0 || (uint32_t)page[u] >= d.num_pages;          // out of sight: behind everything
            if (bad) pool_bad_page(a.pool);
            const size_t at = (size_t)(bad ? 0 : page[u]) * d.kv_heads + h;
            const uint32_t *k = reinterpret_cast<const uint32_t *>(a.pool.block_keys + at * HD) + sub * W;
            if constexpr (W == 4) {
                const uint4 x = __ldcg(reinterpret_cast<const uint4 *>(k));
                key[u][0] = x.x; key[u][1] = x.y; key[u][2] = x.z; key[u][3] = x.w;
            } else {
                const uint2 x = __ldcg(reinterpret_cast<const uint2 *>(k));
                key[u][0] = x.x; key[u][1] = x.y;
            }
            const float s = __ldcg(a.pool.block_key_scales + at);
            scale[u] = bad ? __uint_as_float(0x7FC00000u) : s;
        }
    };
    ask(from + warp * 4);
    // the head's queries, a warp each, to shared memory; their sum in the order of the heads
    for (uint32_t g0 = 0; g0 < group; g0 += SEL_WARPS) {
        if (g0 > 0) __syncthreads();
        if (g0 + warp < group && lane < HD / 8) {
            Row8 x;
            float y[8];
            x.ask(a.q, t * a.q.token_stride + (h * group + g0 + warp) * a.q.head_stride + lane * 8);
            x.values(a.q.type, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) s_rows[warp][lane * 8 + i] = y[i];
        }
        __syncthreads();
        if (tid < HD) {
            float v = g0 == 0 ? s_rows[0][tid] : __fadd_rn(s_sum[tid], s_rows[0][tid]);
            for (uint32_t g = 1; g < min(SEL_WARPS, group - g0); ++g) v = __fadd_rn(v, s_rows[g][tid]);
            s_sum[tid] = v;
        }
    }
    __syncthreads();
    if (warp == 0) {
        constexpr uint32_t LANES = HD / 8;
        const uint32_t l = lane % LANES;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = s_sum[l * 8 + i];
        transform8(v, signs8(a.pool, l * 8), lane);
        uint32_t c[8];
        float unused;
        quantise8<LANES>(v, c, unused);
        if (lane < LANES) *reinterpret_cast<uint2 *>(s_q + l * 8) = make_uint2(four_bytes(c[0], c[1], c[2], c[3]), four_bytes(c[4], c[5], c[6], c[7]));
    }
    __syncthreads();
    int q[W];
#pragma unroll
    for (uint32_t j = 0; j < W; ++j) q[j] = reinterpret_cast<const int *>(s_q)[sub * W + j];
    for (uint32_t i0 = from + warp * 4; i0 < to; i0 += AHEAD * SEL_WARPS * 4) {
        if (i0 != from + warp * 4) ask(i0);
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u) {
            const uint32_t i = i0 + u * SEL_WARPS * 4 + lane / 8;
            int dot = 0;
#pragma unroll
            for (uint32_t j = 0; j < W; ++j) dot = dp4a_ss(key[u][j], q[j], dot);
#pragma unroll
            for (int m = 4; m > 0; m >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, m);
            if (i < to && sub == 0) s_key[i - from] = ordered(__fmul_rn((float)dot, scale[u]));
        }
    }
    __syncthreads();
    const uint32_t m = to - from;
    uint32_t want = a.top - a.sinks - a.local, low = 0;          // keys above `low` are in; of its equals the first `want`
    for (uint32_t i = tid; i < a.sinks; i += SEL_THREADS) out[i] = (int32_t)i;
    for (uint32_t i = tid; i < a.local; i += SEL_THREADS) out[a.top - a.local + i] = (int32_t)(to + i);
    if (want == 0) return;
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {               // byte by byte the key that is the last one wanted
        for (uint32_t i = tid; i < 256; i += SEL_THREADS) s_hist[i] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
        for (uint32_t i = tid; i < m; i += SEL_THREADS)
            if (((s_key[i] ^ low) & mask) == 0) atomicAdd(s_hist + (s_key[i] >> shift & 255u), 1u);
        __syncthreads();
        if (warp == 0) {              // the bin that holds it, from the top
            uint32_t sum = 0, mine[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) { mine[k] = s_hist[255 - (lane * 8 + k)]; sum += mine[k]; }
            uint32_t upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= (uint32_t)o) upto += x; }
            uint32_t before = upto - sum;
            if (before < want && want <= upto)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (before < want && want <= before + mine[k]) { s_pick[0] = 255 - (lane * 8 + k); s_pick[1] = want - before; s_pick[2] = mine[k]; }
                    before += mine[k];
                }
        }
        __syncthreads();
        low |= s_pick[0] << shift;
        want = s_pick[1];
        if (want == s_pick[2]) break;          // the whole bin: everything from its lowest key on
    }
    // in the order of the pages: two scans over the CTA by ballots a stretch
    const bool all_equal = want == s_pick[2];
    uint32_t done = a.sinks, equal = 0, step = 0;
    for (uint32_t i0 = 0; i0 < m; i0 += SEL_THREADS) {
        const uint32_t i = i0 + tid, key = i < m ? s_key[i] : 0;
        const bool tie = !all_equal && i < m && key == low;
        uint32_t eq_before = equal;
        if (!all_equal) {
            const uint32_t e = __ballot_sync(0xffffffffu, tie);
            if (lane == 0) s_warp[step & 1u][warp] = __popc(e);
            __syncthreads();
            for (uint32_t k = 0; k < SEL_WARPS; ++k) {
                if (k < warp) eq_before += s_warp[step & 1u][k];
                equal += s_warp[step & 1u][k];
            }
            eq_before += __popc(e & ((1u << lane) - 1u));
            ++step;
        }
        const bool take = i < m && key >= low && (!tie || eq_before < want);
        const uint32_t b = __ballot_sync(0xffffffffu, take);
        if (lane == 0) s_warp[step & 1u][warp] = __popc(b);
        __syncthreads();
        uint32_t at = done;
        for (uint32_t k = 0; k < SEL_WARPS; ++k) {
            if (k < warp) at += s_warp[step & 1u][k];
            done += s_warp[step & 1u][k];
        }
        ++step;
        at += __popc(b & ((1u << lane) - 1u));
        if (take) out[at] = (int32_t)(from + i);
    }
}

uint32_t row_ctas(const PoolStoreArgs &a, uint32_t ahead) {
    const uint32_t per = ROW_THREADS * 8 / a.pool.d.head_dim * ahead;
    return (uint32_t)(((uint64_t)a.n_tok * 2 * a.pool.d.kv_heads + per - 1) / per);
}
constexpr uint32_t FEW_WRITTEN = 16, FEW_READ = 3;          // CTAs an SM
bool few_rows(const PoolStoreArgs &a, uint32_t few) { return row_ctas(a, 1) <= few * a.sm_count; }
// r / (2 kv heads) for r below 2^31
PoolStoreArgs divided(PoolStoreArgs a) {
    const uint32_t per = 2 * a.pool.d.kv_heads;
    uint32_t bits = 1;
    while ((1u << bits) < per) ++bits;
    a.rows_mul = (uint32_t)(((1ull << (31 + bits)) + per - 1) / per);
    a.rows_shift = bits - 1;
    return a;
}
template <int HD, int BITS> cudaError_t store_rows(cudaStream_t s, const PoolStoreArgs &a, uint32_t *launched) {
    *launched += 1;
    const cudaError_t e = few_rows(a, FEW_WRITTEN) ? launch_kernel(pool_store_kernel<HD, BITS, 1>, dim3(row_ctas(a, 1)), dim3(ROW_THREADS), 0, s, true, a)
                                      : launch_kernel(pool_store_kernel<HD, BITS, 2>, dim3(row_ctas(a, 2)), dim3(ROW_THREADS), 0, s, true, a);
    if (e != cudaSuccess || !a.pool.d.block_keys) return e;
    const uint64_t warps = ((uint64_t)a.n_tok + 31) / 32 * a.pool.d.kv_heads;
    *launched += 1;
    return launch_kernel(pool_block_key_kernel<HD, BITS>, dim3((unsigned)((warps + ROW_THREADS / 32 - 1) / (ROW_THREADS / 32))), dim3(ROW_THREADS), 0, s, true, a);
}
template <int HD, int BITS> cudaError_t load_rows(cudaStream_t s, const PoolStoreArgs &a, uint32_t *launched) {
    *launched += 1;
    return few_rows(a, FEW_READ) ? launch_kernel(pool_load_kernel<HD, BITS, 1>, dim3(row_ctas(a, 1)), dim3(ROW_THREADS), 0, s, true, a)
                       : launch_kernel(pool_load_kernel<HD, BITS, 2>, dim3(row_ctas(a, 2)), dim3(ROW_THREADS), 0, s, true, a);
}

}  // namespace

cudaError_t launch_pool_store(cudaStream_t s, const PoolStoreArgs &args, uint32_t *launched) {
    const PoolStoreArgs a = divided(args);
    const bool wide = a.pool.d.head_dim == 128, b8 = a.pool.d.bits == 8;
    return wide ? (b8 ? store_rows<128, 8>(s, a, launched) : store_rows<128, 4>(s, a, launched)) : b8 ? store_rows<64, 8>(s, a, launched) : store_rows<64, 4>(s, a, launched);
}
cudaError_t launch_pool_load(cudaStream_t s, const PoolStoreArgs &args, uint32_t *launched) {
    const PoolStoreArgs a = divided(args);
    const bool wide = a.pool.d.head_dim == 128, b8 = a.pool.d.bits == 8;
    return wide ? (b8 ? load_rows<128, 8>(s, a, launched) : load_rows<128, 4>(s, a, launched)) : b8 ? load_rows<64, 8>(s, a, launched) : load_rows<64, 4>(s, a, launched);
}
cudaError_t launch_pool_select(cudaStream_t s, const PoolAttnArgs &a, uint32_t *launched) {
    const size_t smem = (size_t)a.pages_stride * 4;
    const uint32_t pairs = a.n_tok * a.pool.d.kv_heads;
    // by the table's width, which is all that is known here of how long the sequences are; the widest leave room for few small CTAs
    const bool small = a.pages_stride <= 4096 && 2 * pairs >= (a.pages_stride <= 1024 ? 5 : 16) * a.sm_count;
    const auto kernel = a.pool.d.head_dim == 128 ? (small ? pool_select_kernel<128, 128> : pool_select_kernel<128, 512>) : small ? pool_select_kernel<64, 128> : pool_select_kernel<64, 512>;
    const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return e;
    *launched += 1;
    return launch_kernel(kernel, dim3(pairs), dim3(small ? 128 : 512), smem, s, true, a);
}

}  // namespace k2t
