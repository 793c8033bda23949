// Rows of the pool: written (signed transform, quantisation, block keys of full pages), read back, and the choice of pages by block keys.
// The arithmetic of a row is that of the engines' caches (store_hadamard_q8_head*_raw, store_hadamard_q4_head_raw, nf4_nearest_idx,
// src/model/real_llm.rs:8303-8365, 8615-8701), operation by operation in fp32, so codes and scales are the same bits.
#include <algorithm>

#include "k2t_kv_pool.cuh"

namespace k2t {
namespace {

__constant__ float CENTROIDS[16] = {-127.f, -96.f, -75.f, -58.f, -44.f, -31.f, -18.f, -6.f, 6.f, 18.f, 31.f, 44.f, 58.f, 75.f, 96.f, 127.f};
__device__ __forceinline__ uint32_t nearest(float y) {
    const float a = fabsf(y);
    const uint32_t p = a < 37.5f ? (a < 12.0f ? 0u : a < 24.5f ? 1u : 2u) : a < 85.5f ? (a < 51.0f ? 3u : a < 66.5f ? 4u : 5u) : a < 111.5f ? 6u : 7u;
    return y >= 0.0f ? 8u + p : 7u - p;
}
constexpr float SMALLEST = 1.1920929e-07f;       // 8-bit rows up to here are stored as zeros

template <int LANES> __device__ __forceinline__ float max_over(float x) {        // of LANES neighbouring lanes
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, m));
    return x;
}
template <int LANES> __device__ __forceinline__ bool any_over(bool b, uint32_t lane) {
    return (__ballot_sync(0xffffffffu, b) >> (lane & ~(uint32_t)(LANES - 1)) & ((1u << LANES) - 1u)) != 0;
}

// A row over LANES lanes, eight values each, as 8-bit codes: what all quantised rows of 8 bits share.  `scale` is NaN for a row that is
// not finite (its codes are 0).
template <int LANES> __device__ __forceinline__ void quantise8(const float (&v)[8], uint32_t lane, int (&code)[8], float &scale) {
    float top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) { top = fmaxf(top, fabsf(v[i])); bad |= not_finite(v[i]); }
    bad = any_over<LANES>(bad, lane);
    top = max_over<LANES>(top);
    const bool zero = top <= SMALLEST || bad;
    const float inv = zero ? 0.0f : __fdiv_rn(127.0f, top);
#pragma unroll
    for (int i = 0; i < 8; ++i) code[i] = zero ? 0 : __float2int_rn(__fmul_rn(v[i], inv));
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
// head_dim / 8 lanes hold a row.  A warp takes 32 * 8 values: 2 rows of 128 or 4 of 64; rows are numbered (token, keys | values, head).
constexpr uint32_t ROW_THREADS = 256;

template <int HD, int BITS> __global__ void __launch_bounds__(ROW_THREADS) pool_store_kernel(const __grid_constant__ PoolStoreArgs a) {
    using B = PoolBlock<HD, BITS>;
    constexpr uint32_t LANES = HD / 8, PER = 32 / LANES;
    const uint32_t lane = threadIdx.x & 31, l = lane % LANES, kh = a.pool.d.kv_heads;
    const uint64_t r = ((uint64_t)blockIdx.x * (ROW_THREADS / 32) + (threadIdx.x >> 5)) * PER + lane / LANES;
    const bool live = r < (uint64_t)a.n_tok * 2 * kh;
    const uint32_t t = live ? (uint32_t)(r / (2 * kh)) : 0, u = live ? (uint32_t)(r % (2 * kh)) : 0, value = u >= kh ? 1 : 0, head = u - value * kh;
    pdl_wait();
    pdl_trigger();
    uint32_t row = 0;
    uint8_t *block = live ? block_of(a.pool, __ldcg(a.slots + t), head, B::BYTES, row) : nullptr;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const RowsArg &src = value ? a.v : a.k;
    if (block != nullptr) rows_get8(src, t * src.token_stride + head * src.head_stride + l * 8, v);
    transform8(v, signs8(a.pool, l * 8), lane);
    if (BITS == 8) {
        int c[8];
        float scale;
        quantise8<LANES>(v, lane, c, scale);
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i / 4] |= (uint32_t)(c[i] + 128) << (i % 4 * 8);
        if (block == nullptr) return;
        *reinterpret_cast<uint2 *>(block + value * B::V_AT + row_place<B::RB>(row, l * 8)) = make_uint2(w[0], w[1]);
        if (l == 0) reinterpret_cast<float *>(block + (value ? B::VS_AT : B::KS_AT))[row] = scale;
    } else {
        float top = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) { top = fmaxf(top, fabsf(v[i])); bad |= not_finite(v[i]); }
        bad = any_over<LANES>(bad, lane);            // of the whole row: its groups stand or fall together
        top = max_over<8>(top);
        const bool zero = top < 1e-30f || bad;
        const float inv0 = zero ? 0.0f : __fdiv_rn(127.0f, top);
        float rc[8], den = 0.0f, num = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = CENTROIDS[nearest(__fmul_rn(v[i], inv0))];
            rc[i] = __fmul_rn(v[i], c);
            den += c * c;                    // whole numbers below 2^24: in any order
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
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) w |= (zero ? 8u : nearest(__fmul_rn(v[i], inv))) << (4 * i);
        if (block == nullptr) return;
        *reinterpret_cast<uint32_t *>(block + value * B::V_AT + row_place<B::RB>(row, l * 4)) = w;
        if (l % 8 == 0) reinterpret_cast<uint16_t *>(block + (value ? B::VS_AT : B::KS_AT))[row * B::G + l / 8] = bad ? 0x7FC0u : __bfloat16_as_ushort(sb);
    }
}

// Eight stored values of a row, element 8 l on, times their scale.
template <int HD, int BITS> __device__ __forceinline__ void stored8(const uint8_t *block, uint32_t rows_at, uint32_t scales_at, uint32_t row, uint32_t l, float (&v)[8]) {
    using B = PoolBlock<HD, BITS>;
    if (BITS == 8) {
        const uint2 w = __ldcg(reinterpret_cast<const uint2 *>(block + rows_at + row_place<B::RB>(row, l * 8)));
        const float s = __ldcg(reinterpret_cast<const float *>(block + scales_at) + row);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn((float)((int)(((i < 4 ? w.x : w.y) >> (i % 4 * 8)) & 255u) - 128), s);
    } else {
        const uint32_t w = __ldcg(reinterpret_cast<const uint32_t *>(block + rows_at + row_place<B::RB>(row, l * 4)));
        const float s = bf16_bits_to_f32(__ldcg(reinterpret_cast<const uint16_t *>(block + scales_at) + row * B::G + l / 8));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(CENTROIDS[w >> (4 * i) & 15u], s);
    }
}

template <int HD, int BITS> __global__ void __launch_bounds__(ROW_THREADS) pool_load_kernel(const __grid_constant__ PoolStoreArgs a) {
    using B = PoolBlock<HD, BITS>;
    constexpr uint32_t LANES = HD / 8, PER = 32 / LANES;
    const uint32_t lane = threadIdx.x & 31, l = lane % LANES, kh = a.pool.d.kv_heads;
    const uint64_t r = ((uint64_t)blockIdx.x * (ROW_THREADS / 32) + (threadIdx.x >> 5)) * PER + lane / LANES;
    const bool live = r < (uint64_t)a.n_tok * 2 * kh;
    const uint32_t t = live ? (uint32_t)(r / (2 * kh)) : 0, u = live ? (uint32_t)(r % (2 * kh)) : 0, value = u >= kh ? 1 : 0, head = u - value * kh;
    pdl_wait();
    pdl_trigger();
    uint32_t row = 0;
    const uint8_t *block = live ? block_of(a.pool, __ldcg(a.slots + t), head, B::BYTES, row) : nullptr;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (block != nullptr) stored8<HD, BITS>(block, value ? B::V_AT : 0, value ? B::VS_AT : B::KS_AT, row, l, v);
    transform8_back(v, signs8(a.pool, l * 8), lane);
    const RowsArg &dst = value ? a.v : a.k;
    if (block != nullptr) rows_put8(dst, t * dst.token_stride + head * dst.head_stride + l * 8, v);
}

// ------------------------------------------------------------------------------------------------ block keys
// The mean of a page's keys as they are stored (transformed), summed in the order of their positions, quantised as an 8-bit row.  The
// token that writes a page's last row makes it.  A warp looks over 32 tokens of a head.
template <int HD, int BITS> __global__ void __launch_bounds__(ROW_THREADS) pool_block_key_kernel(const __grid_constant__ PoolStoreArgs a) {
    using B = PoolBlock<HD, BITS>;
    constexpr uint32_t LANES = HD / 8;
    const uint32_t lane = threadIdx.x & 31, l = lane % LANES, kh = a.pool.d.kv_heads, pt = 1u << a.pool.d.page_shift;
    const uint64_t w = (uint64_t)blockIdx.x * (ROW_THREADS / 32) + (threadIdx.x >> 5);
    const uint32_t head = (uint32_t)(w % kh);
    const uint64_t t = w / kh * 32 + lane;
    pdl_wait();
    pdl_trigger();
    const int64_t slot = t < a.n_tok ? __ldcg(a.slots + t) : -1;
    const bool last = slot >= 0 && ((uint32_t)slot & (pt - 1)) == pt - 1 && (uint64_t)slot >> a.pool.d.page_shift < a.pool.d.num_pages;
    for (uint32_t todo = __ballot_sync(0xffffffffu, last); todo != 0; todo &= todo - 1) {
        const uint64_t page = (uint64_t)__shfl_sync(0xffffffffu, slot, __ffs(todo) - 1) >> a.pool.d.page_shift;
        const uint8_t *block = a.pool.rows + ((page * kh + head) << (a.pool.d.page_shift - 4)) * B::BYTES;
        float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 8
        for (uint32_t i = 0; i < pt; ++i) {
            float v[8];
            stored8<HD, BITS>(block + (size_t)(i >> 4) * B::BYTES, 0, B::KS_AT, i & 15u, l, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum[k] = __fadd_rn(sum[k], v[k]);
        }
        const float part = 1.0f / (float)pt;             // a power of two
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] = __fmul_rn(sum[k], part);
        int c[8];
        float scale;
        quantise8<LANES>(sum, lane, c, scale);
        uint32_t word[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < 8; ++k) word[k / 4] |= ((uint32_t)c[k] & 255u) << (k % 4 * 8);
        if (lane < LANES) *reinterpret_cast<uint2 *>(a.pool.block_keys + (page * kh + head) * HD + l * 8) = make_uint2(word[0], word[1]);
        if (lane == 0) a.pool.block_key_scales[page * kh + head] = scale;
    }
}

// ------------------------------------------------------------------------------------------------ choice of pages
// CTA = (token, kv head).  The query is the sum of the head's queries, quantised as an 8-bit row; a page scores the whole-number product
// with its block key times the key's scale (one rounding, so that scores are the same wherever they are computed).  The order of
// scores is that of their bits as numbers; the highest `want` of them are found by four passes over their bytes, ties by index.
// Two sizes of CTA: with few (token, kv head) pairs the time is one CTA's chain of loads, and 512 threads have a whole sequence's keys in
// flight; with many, smaller CTAs have fewer threads idle at their barriers.
__device__ __forceinline__ uint32_t ordered(float x) {           // NaN behind everything
    if (x != x) return 0;
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <int HD, uint32_t SEL_THREADS> __global__ void __launch_bounds__(SEL_THREADS) pool_select_kernel(const __grid_constant__ PoolAttnArgs a) {
    constexpr uint32_t SEL_WARPS = SEL_THREADS / 32;
    extern __shared__ uint32_t s_key[];
    __shared__ __align__(16) int8_t s_q[HD];
    __shared__ uint32_t s_hist[256], s_warp[SEL_WARPS], s_pick[2];
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
            const bool bad = page[u] < 0 || (uint32_t)page[u] >= d.num_pages;          // scores 0
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
            scale[u] = bad ? 0.0f : s;
        }
    };
    ask(from + warp * 4);
    if (warp == SEL_WARPS - 1) {
        constexpr uint32_t LANES = HD / 8;
        const uint32_t l = lane % LANES;
        float v[8];
#pragma unroll 1
        for (uint32_t g0 = 0; g0 < group; g0 += 8) {          // the sum in the order of the heads, eight of them on their way
            float x[8][8];
#pragma unroll
            for (uint32_t g = 0; g < 8; ++g)
                if (g0 + g < group) rows_get8(a.q, t * a.q.token_stride + (h * group + g0 + g) * a.q.head_stride + l * 8, x[g]);
#pragma unroll
            for (uint32_t g = 0; g < 8; ++g)
                if (g0 + g < group)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = g0 + g == 0 ? x[g][i] : __fadd_rn(v[i], x[g][i]);
        }
        transform8(v, signs8(a.pool, l * 8), lane);
        int c[8];
        float unused;
        quantise8<LANES>(v, lane, c, unused);
        if (lane < LANES)
#pragma unroll
            for (int i = 0; i < 8; ++i) s_q[l * 8 + i] = (int8_t)c[i];
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
    uint32_t want = a.top - a.sinks - a.local, prefix = 0;         // keys above `prefix` are in; of its equals the first `want`
    if (want > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (uint32_t i = tid; i < 256; i += SEL_THREADS) s_hist[i] = 0;
            __syncthreads();
            const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
            for (uint32_t i = tid; i < m; i += SEL_THREADS)
                if (((s_key[i] ^ prefix) & mask) == 0) atomicAdd(s_hist + (s_key[i] >> shift & 255u), 1u);
            __syncthreads();
            if (warp == 0) {              // the bin that holds the last one wanted, from the top
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
                        if (before < want && want <= before + mine[k]) { s_pick[0] = 255 - (lane * 8 + k); s_pick[1] = want - before; }
                        before += mine[k];
                    }
            }
            __syncthreads();
            prefix |= s_pick[0] << shift;
            want = s_pick[1];
            __syncthreads();
        }
    } else {
        prefix = 0xFFFFFFFFu;             // above every score
    }
    // in the order of the pages: sinks, the chosen ones, the last ones
    for (uint32_t i = tid; i < a.sinks; i += SEL_THREADS) out[i] = (int32_t)i;
    for (uint32_t i = tid; i < a.local; i += SEL_THREADS) out[a.top - a.local + i] = (int32_t)(to + i);
    uint32_t done = a.sinks, equal = 0;
    for (uint32_t i0 = 0; i0 < m; i0 += SEL_THREADS) {
        const uint32_t i = i0 + tid, key = i < m ? s_key[i] : 0;
        const bool is_equal = i < m && key == prefix;
        // counts of equals before this one, then of takers: two scans over the CTA by ballots
        const uint32_t e = __ballot_sync(0xffffffffu, is_equal);
        if (lane == 0) s_warp[warp] = __popc(e);
        __syncthreads();
        uint32_t eq_before = equal, eq_all = 0;
        for (uint32_t k = 0; k < SEL_WARPS; ++k) {
            if (k < warp) eq_before += s_warp[k];
            eq_all += s_warp[k];
        }
        eq_before += __popc(e & ((1u << lane) - 1u));
        __syncthreads();
        const bool take = i < m && (key > prefix || (is_equal && eq_before < want));
        const uint32_t b = __ballot_sync(0xffffffffu, take);
        if (lane == 0) s_warp[warp] = __popc(b);
        __syncthreads();
        uint32_t at = done, all = 0;
        for (uint32_t k = 0; k < SEL_WARPS; ++k) {
            if (k < warp) at += s_warp[k];
            all += s_warp[k];
        }
        at += __popc(b & ((1u << lane) - 1u));
        if (take) out[at] = (int32_t)(from + i);
        __syncthreads();
        done += all;
        equal += eq_all;
    }
}

template <int HD, int BITS> cudaError_t store_rows(cudaStream_t s, const PoolStoreArgs &a, uint32_t *launched) {
    const uint64_t rows = (uint64_t)a.n_tok * 2 * a.pool.d.kv_heads, per = ROW_THREADS * 8 / HD, warps = ((uint64_t)a.n_tok + 31) / 32 * a.pool.d.kv_heads;
    *launched += 1;
    const cudaError_t e = launch_kernel(pool_store_kernel<HD, BITS>, dim3((unsigned)((rows + per - 1) / per)), dim3(ROW_THREADS), 0, s, true, a);
    if (e != cudaSuccess || !a.pool.d.block_keys) return e;
    *launched += 1;
    return launch_kernel(pool_block_key_kernel<HD, BITS>, dim3((unsigned)((warps + ROW_THREADS / 32 - 1) / (ROW_THREADS / 32))), dim3(ROW_THREADS), 0, s, true, a);
}
template <int HD, int BITS> cudaError_t load_rows(cudaStream_t s, const PoolStoreArgs &a, uint32_t *launched) {
    const uint64_t rows = (uint64_t)a.n_tok * 2 * a.pool.d.kv_heads, per = ROW_THREADS * 8 / HD;
    *launched += 1;
    return launch_kernel(pool_load_kernel<HD, BITS>, dim3((unsigned)((rows + per - 1) / per)), dim3(ROW_THREADS), 0, s, true, a);
}

}  // namespace

cudaError_t launch_pool_store(cudaStream_t s, const PoolStoreArgs &a, uint32_t *launched) {
    const bool wide = a.pool.d.head_dim == 128, b8 = a.pool.d.bits == 8;
    return wide ? (b8 ? store_rows<128, 8>(s, a, launched) : store_rows<128, 4>(s, a, launched)) : b8 ? store_rows<64, 8>(s, a, launched) : store_rows<64, 4>(s, a, launched);
}
cudaError_t launch_pool_load(cudaStream_t s, const PoolStoreArgs &a, uint32_t *launched) {
    const bool wide = a.pool.d.head_dim == 128, b8 = a.pool.d.bits == 8;
    return wide ? (b8 ? load_rows<128, 8>(s, a, launched) : load_rows<128, 4>(s, a, launched)) : b8 ? load_rows<64, 8>(s, a, launched) : load_rows<64, 4>(s, a, launched);
}
cudaError_t launch_pool_select(cudaStream_t s, const PoolAttnArgs &a, uint32_t *launched) {
    const size_t smem = (size_t)a.pages_stride * 4;
    const uint32_t pairs = a.n_tok * a.pool.d.kv_heads;
    const bool small = pairs >= 4 * a.sm_count && a.pages_stride <= 4096;
    const auto kernel = a.pool.d.head_dim == 128 ? (small ? pool_select_kernel<128, 128> : pool_select_kernel<128, 512>) : small ? pool_select_kernel<64, 128> : pool_select_kernel<64, 512>;
    const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return e;
    *launched += 1;
    return launch_kernel(kernel, dim3(pairs), dim3(small ? 128 : 512), smem, s, true, a);
}

}  // namespace k2t
