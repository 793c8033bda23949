// Attention of many query rows over the pages of a shared prefix: the rows of all tokens against the same keys and values, on the
// tensor-memory cores.  The mathematics is that of k2t_pool_attn.cu (weights that carry the values' scales, codes as exact halves).
//   * A CTA takes a stretch of an item of the prefix in tiles of 64 positions, as two STREAMS of 128 rows: an item is a kv head and 256 rows,
//     or, where there are no more than 128 or a row has two terms (their operands would not fit), 128 rows, whose even and odd tiles are
//     the streams.  While the softmax warps of one stream work, the products of the other run.
//   * One warp asks for the blocks of a tile (bulk copies into a ring of raw tiles; as loads into registers, two tiles in flight, they were
//     throttled by the little L1 that the operands leave: 2200 cycles a tile).  Four warps expand the codes to halves in the operand layout
//     (panels of 64 columns, 128-byte rows, 128-byte swizzle) and the tile's scales to column constants.
//   * One warp issues S = Q K^T (queries from shared memory) and O += P V (weights from tensor memory, where they overwrite S).  All its lanes
//     run along and an elected one issues, which keeps descriptors in uniform registers: as a branch of lane 0, or with a predicate of lanes,
//     a product took 75 (scores) and 97 cycles to issue and was the bound (160 sequences behind 32768 positions 323 us, 286 elected).
//   * Eight warps of softmax read S in fragments of 16x256b: a lane then has 4 rows and a quarter of the columns, so that it reads a quarter
//     of the column constants; O is rescaled only where a row's maximum has grown by 2^8 or more.
// The tiles of all items form one line that is cut into equal parts, one per CTA; partial results are joined by pool_merge_kernel.
#include "k2t_flash_tc.cuh"
#include "k2t_kv_pool.cuh"
#include "k2t_pool_attn.h"

namespace k2t {
namespace {

constexpr uint32_t FL_KT = 64, FL_SOFT = 8, FL_CONV = 4, FL_ISSUE = FL_SOFT + FL_CONV, FL_LOAD = FL_ISSUE + 1, FL_THREADS = (FL_LOAD + 1) * 32, FL_WAIT = 1u << 22, FL_COLS = 512;

template <int HD, int BITS, int QT> struct Flash {
    using B = PoolBlock<HD, BITS>;
    // two groups of 64 elements a row: with queries and weights of one half the groups' scales go into the codes, relative to the larger one (a
    // rounding to 11 bits, like that of the queries); with two, each group has scores, weights and products of its own
    static constexpr bool FOLD = B::G == 2 && QT == 1;
    static constexpr uint32_t PD = HD / 64, G = FOLD ? 1 : B::G, STAGES = HD == 128 && BITS == 8 ? 3 : 4, RAWS = 3, BLOCKS = FL_KT / POOL_ROWS;          // what shared memory holds
    static constexpr uint32_t Q_TILE = PD * FLASH_ROWS * 128, K_TILE = PD * FL_KT * 128, RAW = (BLOCKS * B::BYTES + 127) / 128 * 128, CONST = G == 1 ? 24 : 48;        // bytes; CONST per pair of columns
    static constexpr uint32_t CONSTS = 1024, HEAD = (CONSTS + STAGES * (FL_KT / 2) * CONST + 1023) / 1024 * 1024;
    static constexpr uint32_t Q_AT = HEAD, K_AT = Q_AT + 2 * Q_TILE, RAW_AT = K_AT + STAGES * 2 * K_TILE, SMEM = RAW_AT + RAWS * RAW + 1024;          // two tiles of queries: of rows, or of terms
};

using u64 = unsigned long long;
__device__ __forceinline__ u64 pair_of(uint32_t lo, uint32_t hi) { u64 d; asm("mov.b64 %0, {%1,%2};" : "=l"(d) : "r"(lo), "r"(hi)); return d; }
__device__ __forceinline__ u64 pair_of(float lo, float hi) { return pair_of(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ void unpair(u64 p, float &lo, float &hi) { uint32_t a, b; asm("mov.b64 {%0,%1}, %2;" : "=r"(a), "=r"(b) : "l"(p)); lo = __uint_as_float(a); hi = __uint_as_float(b); }
__device__ __forceinline__ u64 mul2(u64 a, u64 b) { u64 d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ u64 add2(u64 a, u64 b) { u64 d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) { u64 d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }
__device__ __forceinline__ void lds_pairs(uint32_t at, u64 &x, u64 &y) { asm volatile("ld.shared.v2.b64 {%0,%1}, [%2];" : "=l"(x), "=l"(y) : "r"(at)); }
__device__ __forceinline__ u64 lds_pair(uint32_t at) { u64 x; asm volatile("ld.shared.b64 %0, [%1];" : "=l"(x) : "r"(at)); return x; }

__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }

// 16 lanes of tensor memory in fragments: word 4 i + 2 k + e of a thread is row lane / 4 + 8 k, column 8 i + 2 (lane % 4) + e
__device__ __forceinline__ void tm_ld_frag64(uint32_t taddr, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : K2T_R8(v, 0), K2T_R8(v, 8), K2T_R8(v, 16), K2T_R8(v, 24) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tm_ld_frag32(uint32_t taddr, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];" : K2T_R8(v, 0), K2T_R8(v, 8) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tm_st_frag32(uint32_t taddr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::K2T_I8(v, 0), K2T_I8(v, 8), "r"(taddr) : "memory");
}
// 32 words of 16 lanes: word 2 i + k of a thread is row lane / 4 + 8 k, column 4 i + lane % 4
__device__ __forceinline__ void tm_st_words32(uint32_t taddr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::K2T_I8(v, 0), K2T_I8(v, 8), "r"(taddr) : "memory");
}
__device__ __forceinline__ void sts4(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// One lane of a warp that is together, always the same one.
__device__ __forceinline__ bool elected() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ uint4 lds4(uint32_t at) { uint4 v; asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at)); return v; }
__device__ __forceinline__ uint32_t lds1(uint32_t at) { uint32_t v; asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at)); return v; }

struct Segment { uint32_t item, first, last; };          // tiles [first, last) of an item
// Segment s of a CTA's part of the line; false behind the last.
__device__ __forceinline__ bool segment_of(const FlashArgs &f, uint32_t s, Segment &g) {
    const uint32_t x0 = blockIdx.x * f.part, x1 = min(f.items * f.tiles, x0 + f.part);          // below 2^32: see MOST_TILES
    const uint32_t item = x0 / f.tiles + s, b = item * f.tiles;
    if (b >= x1) return false;
    g.item = item;
    g.first = x0 > b ? x0 - b : 0;
    g.last = min(f.tiles, x1 - b);
    return true;
}

// ------------------------------------------------------------------------------------------------ tiles
// Where the 16-byte unit (r, c) of a block's 16 rows lies in the rows: the inverse of row_place.
template <uint32_t RB> __device__ __forceinline__ void unit_place(uint32_t r, uint32_t c, uint32_t &row, uint32_t &chunk) {
    const uint32_t quad = (r >> 2) & 3u;
    row = RB == 128 ? r : RB == 64 ? r ^ (quad & 1u) : r ^ ((quad >> 1) | ((quad & 1u) << 1));
    chunk = RB == 128 ? c ^ ((quad << 1) ^ ((r & 1u) << 2)) : RB == 64 ? c ^ (2u * ((quad ^ (quad >> 1)) & 1u)) : c;
}

// 128 threads.  A thread has the same unit of 16 bytes in every block it reads (a block of keys or values has RB units: one per thread, or
// a thread reads every second or fourth block), so what it does to a block is loads and stores at fixed distances.
template <int HD, int BITS, int QT> struct Converter {
    using B = PoolBlock<HD, BITS>;
    using F = Flash<HD, BITS, QT>;
    static constexpr uint32_t STEP = 128 / B::RB, PER = F::BLOCKS / STEP;          // blocks between two of a thread; of a thread
    static_assert(FL_CONV == 4, "128 threads");
    uint32_t ct, first, load_at, store_at, store_x, row_in;
    bool second;                 // of the row's two groups
    Expand ex;

    __device__ __forceinline__ explicit Converter(uint32_t thread) : ct(thread) {
        // eight neighbouring threads: four chunks of two neighbouring rows, whose stores meet in no bank (rows differ in the last bit of the swizzle)
        const uint32_t u = ct % B::RB;
        first = ct / B::RB;
        uint32_t r, c;
        if (B::RB == 128) { c = (u & 3u) | (u >> 1 & 4u); r = (u >> 2 & 1u) | (u >> 4) << 1; }
        else { c = u % (B::RB / 16); r = u / (B::RB / 16); }
        load_at = (r * (B::RB / 16) + c) * 16;
        uint32_t row, chunk;
        unit_place<B::RB>(r, c, row, chunk);
        const uint32_t c0 = BITS == 8 ? chunk * 2 : chunk * 4;          // first 16-byte chunk of halves
        store_at = (c0 >> 3) * (FL_KT * 128) + row * 128;
        store_x = (c0 & 7u) ^ (row & 7u);
        row_in = row;
        second = c0 >= 8;
    }
    static constexpr bool SCALED = BITS == 4 && F::G == 1;          // values of 4 bits whose weights have no factor per group
    template <bool FACTOR> __device__ __forceinline__ void expand(uint32_t at, const uint4 &w, uint32_t factor) const {          // `at`: the thread's row and panel
        if (BITS == 8) {
            sts4(at + (store_x << 4), ex.halves_lo(w.x), ex.halves_hi(w.x), ex.halves_lo(w.y), ex.halves_hi(w.y));
            sts4(at + ((store_x ^ 1u) << 4), ex.halves_lo(w.z), ex.halves_hi(w.z), ex.halves_lo(w.w), ex.halves_hi(w.w));
        } else {
            const uint32_t x[4] = {w.x, w.y, w.z, w.w};
            auto scaled = [&](uint32_t h) {
                if (!FACTOR) return h;
                const __half2 y = __hmul2(*reinterpret_cast<const __half2 *>(&h), *reinterpret_cast<const __half2 *>(&factor));
                return *reinterpret_cast<const uint32_t *>(&y);
            };
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t lo = ex.centroids4(x[i]), hi = ex.centroids4(x[i] >> 16);
                sts4(at + ((store_x ^ i) << 4), scaled(ex.halves_lo(lo)), scaled(ex.halves_hi(lo)), scaled(ex.halves_lo(hi)), scaled(ex.halves_hi(hi)));
            }
        }
    }
    // The thread's group's scale over the one that the row has in its column's constants (the larger one; of values weight_scale of it), in both
    // halves; 0 for a row of zeros and one that is out of sight or not finite.  Of a single group 1, or 0 and little more.
    __device__ __forceinline__ uint32_t factor_of(uint32_t scales, bool seen, bool value) const {
        const float a = __uint_as_float(scales << 16), b = __uint_as_float(scales & 0xFFFF0000u), mine = (F::FOLD ? second : (row_in & 1u) != 0) ? b : a, top = F::FOLD ? fmaxf(a, b) : mine;
        const float x = seen && top > 0.0f ? mine * rcp_approx(value ? weight_scale(top) : top) : 0.0f;
        return half2_bits(x, x);
    }
    // A raw tile at shared address `raw` becomes an operand tile; in sight are the first `end` positions of blocks with their bit set.
    __device__ __forceinline__ void put(uint32_t raw, uint32_t s_tile, uint8_t *consts, uint32_t blocks, uint32_t end) const {
        const bool seen = (blocks >> (ct / POOL_ROWS % F::BLOCKS) & 1u) != 0 && ct < end;
        uint4 k[PER], v[PER];
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) k[i] = lds4(raw + (first + i * STEP) * B::BYTES + load_at);
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) v[i] = lds4(raw + (first + i * STEP) * B::BYTES + B::V_AT + load_at);
        uint32_t kf[PER], vf[PER];
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            kf[i] = vf[i] = 0;
            if (SCALED) {
                const uint32_t b = first + i * STEP, at = raw + b * B::BYTES + (row_in * B::G & ~1u) * 2;          // one row's two groups, or two rows
                const bool there = (blocks >> b & 1u) != 0 && b * POOL_ROWS + row_in < end;
                if (F::FOLD) kf[i] = factor_of(lds1(at + B::KS_AT), there, false);
                vf[i] = factor_of(lds1(at + B::VS_AT), there, true);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) expand<F::FOLD>(s_tile + store_at + (first + i * STEP) * (POOL_ROWS * 128), k[i], kf[i]);
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) expand<SCALED>(s_tile + F::K_TILE + store_at + (first + i * STEP) * (POOL_ROWS * 128), v[i], vf[i]);
        if (ct < FL_KT) {
            constexpr uint32_t G = F::G;
            const uint32_t at = raw + ct / POOL_ROWS * B::BYTES, row = ct % POOL_ROWS;
            float ks[2], vs[2], lv = -INFINITY, iv = 0.0f, part[2] = {0.0f, 0.0f};
            if (BITS == 8) {
                ks[0] = __uint_as_float(lds1(at + B::KS_AT + row * 4));
                vs[0] = __uint_as_float(lds1(at + B::VS_AT + row * 4));
            } else {
                const uint32_t a = lds1(at + B::KS_AT + (row * B::G & ~1u) * 2), b = lds1(at + B::VS_AT + (row * B::G & ~1u) * 2);          // one row's two groups, or two rows
                const bool high = B::G == 1 && (row & 1u);
                ks[0] = __uint_as_float(high ? a & 0xFFFF0000u : a << 16); ks[1] = __uint_as_float(a & 0xFFFF0000u);
                vs[0] = __uint_as_float(high ? b & 0xFFFF0000u : b << 16); vs[1] = __uint_as_float(b & 0xFFFF0000u);
                if (F::FOLD) {                 // the larger one; all groups of a row are NaN or none
                    ks[0] = fmaxf(ks[0], ks[1]);
                    vs[0] = fmaxf(vs[0], vs[1]);
                }
            }
            if (seen) {
                const float u = weight_scale(G == 1 ? vs[0] : fmaxf(vs[0], vs[1]));          // of zeros 8-bit codes are 0, 4-bit ones have factors
                lv = log2_approx(u);
                iv = rcp_approx(u);
#pragma unroll
                for (uint32_t g = 0; g < G; ++g) part[g] = vs[g] * iv;
            } else {
                ks[0] = ks[1] = 0.0f;
            }
            float *c = reinterpret_cast<float *>(consts);
            const uint32_t i = ct >> 1, e = ct & 1u;
            if (G == 1) {
                c[4 * i + e] = ks[0];
                c[4 * i + 2 + e] = lv;
                c[4 * (FL_KT / 2) + 2 * i + e] = iv;
            } else {
                c[12 * i + e] = ks[0];
                c[12 * i + 2 + e] = ks[1];
                c[12 * i + 4 + e] = lv;
                c[12 * i + 6 + e] = iv;
                c[12 * i + 8 + e] = part[0];
                c[12 * i + 10 + e] = part[1];
            }
        }
    }
};

// ------------------------------------------------------------------------------------------------ queries
// The rows of all items as the kernel's first operand, made once for all parts of the line: transformed, scaled by a power of two, one or two
// halves, in the layout of shared memory ([item][tile of 128 rows][term][panel][row]: a bulk copy brings a tile); their factors behind them.
constexpr uint32_t QK_THREADS = 256;
template <int HD, int QT> __global__ void __launch_bounds__(QK_THREADS) pool_query_kernel(const __grid_constant__ SplitArgs p) {
    constexpr uint32_t LANES = HD / 8, TILE = HD / 64 * FLASH_ROWS * 128;
    const FlashArgs &f = p.flash;
    const uint32_t lane = threadIdx.x & 31u, l = lane % LANES, group = p.a.heads / p.a.pool.d.kv_heads, all = p.a.n_tok * group;
    const uint32_t per = (f.halved ? 1 : 2) * FLASH_ROWS, at = (blockIdx.x * QK_THREADS + threadIdx.x) / LANES, item = at / per, row = at % per;          // whole warps below the last item
    pdl_wait();
    pdl_trigger();
    const uint32_t h = item / f.row_tiles, r = item % f.row_tiles * per + row;
    if (item >= f.items) return;
    uint32_t hi[4], lo[4];
    const float down = query_halves<HD>(p.a.pool, p.a.q, r < all, r / group * p.a.q.token_stride + (h * group + r % group) * p.a.q.head_stride, l, lane, hi, lo);
    if (l == 0) f.factors[item * per + row] = p.a.scale * LOG2E * down;
    uint8_t *to = f.queries + ((size_t)item * (per / FLASH_ROWS) + row / FLASH_ROWS) * QT * TILE + (l / 8) * (FLASH_ROWS * 128) + row % FLASH_ROWS * 128 + (((l % 8) ^ (row & 7u)) << 4);
    *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (QT == 2) *reinterpret_cast<uint4 *>(to + TILE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

template <int HD, int BITS, int QT, int PT>
__global__ void __launch_bounds__(FL_THREADS, 1) pool_flash_kernel(const __grid_constant__ SplitArgs p) {
    using F = Flash<HD, BITS, QT>;
    constexpr uint32_t G = F::G, STAGES = F::STAGES;
    static_assert(STAGES >= 3, "tiles in use at a time, see the order of the products");
    extern __shared__ uint8_t smem_raw[];
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw), sbase = (raw + 1023u) & ~1023u;
    uint8_t *smem = smem_raw + (sbase - raw);
    const FlashArgs &f = p.flash;
    // barriers: tiles ready / free; of each stream: S ready (two buffers), weights ready (two), O updated; queries; end of a segment; end; raw
    // tiles landed / free
    const uint32_t b_full = sbase, b_free = b_full + 8 * STAGES, b_s = b_free + 8 * STAGES, b_p = b_s + 32, b_o = b_p + 32, b_q = b_o + 16, b_end = b_q + 8, b_last = b_end + 8, b_rfull = b_last + 8, b_rfree = b_rfull + 8 * F::RAWS;
    volatile uint32_t *s_tmem = reinterpret_cast<volatile uint32_t *>(smem + 512), *s_abort = reinterpret_cast<volatile uint32_t *>(smem + 516);
    const uint32_t s_q = sbase + F::Q_AT, s_k = sbase + F::K_AT, s_raw = sbase + F::RAW_AT;
    if (tid == 0) {
        for (uint32_t i = 0; i < STAGES; ++i) { mbar_init(b_full + 8 * i, FL_CONV); mbar_init(b_free + 8 * i, 1); }
        for (uint32_t i = 0; i < 4; ++i) { mbar_init(b_s + 8 * i, 1); mbar_init(b_p + 8 * i, 128); }
        for (uint32_t i = 0; i < 2; ++i) mbar_init(b_o + 8 * i, 1);
        mbar_init(b_q, 1);
        mbar_init(b_end, 1);
        mbar_init(b_last, 1);
        for (uint32_t i = 0; i < F::RAWS; ++i) { mbar_init(b_rfull + 8 * i, 1); mbar_init(b_rfree + 8 * i, FL_CONV); }
        *s_abort = 0;
        fence_mbar_init();
    }
    if (warp == FL_ISSUE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sbase + 512), "r"(FL_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    pdl_wait();
    pdl_trigger();
    // tensor memory of a stream: 128 columns of S (two buffers, or a tile's two groups of 64 elements), HD columns of O
    const uint32_t t_stream = 128 + HD;
    Segment g;
    bool ok = true;

    if (warp == FL_LOAD) {
        // lane b asks for block b of a tile; a raw tile holds the blocks as they lie
        const PoolShape &d = p.a.pool.d;
        uint32_t n = 0;
        for (uint32_t s = 0; ok && segment_of(f, s, g); ++s) {
            const uint32_t head = g.item / f.row_tiles;
            auto page_of = [&](uint32_t tile) {
                const uint32_t pos = tile * FL_KT + lane * POOL_ROWS;
                return lane < F::BLOCKS && tile < g.last && pos < p.a.prefix_len ? __ldcg(p.a.prefix_pages + (pos >> d.page_shift)) : 0;
            };
            int32_t page = page_of(g.first);
            for (uint32_t t = g.first; t < g.last; ++t, ++n) {
                const uint32_t slot = n % F::RAWS, pos = t * FL_KT + lane * POOL_ROWS;
                const int32_t next = page_of(t + 1);
                if (n >= F::RAWS) ok = mbar_wait_warp(b_rfree + 8 * slot, (n / F::RAWS - 1) & 1u, FL_WAIT, s_abort);
                if (!ok) break;
                const bool there = lane < F::BLOCKS && pos < p.a.prefix_len, good = there && page >= 0 && (uint32_t)page < d.num_pages;
                if (there && !good) pool_bad_page(p.a.pool);
                const uint32_t blocks = __ballot_sync(0xffffffffu, good);
                if (lane == 0) {
                    reinterpret_cast<volatile uint32_t *>(smem + 528)[slot] = blocks;          // which of the tile's blocks are in sight
                    mbar_expect_tx(b_rfull + 8 * slot, __popc(blocks) * F::B::BYTES);
                }
                __syncwarp();
                if (good)
                    bulk_g2s(s_raw + slot * F::RAW + lane * F::B::BYTES,
                             p.a.pool.rows + ((((size_t)page * d.kv_heads + head) << (d.page_shift - 4)) + ((pos & ((1u << d.page_shift) - 1u)) >> 4)) * F::B::BYTES, F::B::BYTES, b_rfull + 8 * slot);
                page = next;
            }
        }
        // the copies in flight land before the CTA leaves, also after a wait that gave up
        for (uint32_t i = n > F::RAWS ? n - F::RAWS : 0; i < n; ++i)
            for (uint32_t spin = 0; spin < FL_WAIT && !mbar_try_wait(b_rfull + 8 * (i % F::RAWS), (i / F::RAWS) & 1u); ++spin) {}
    } else if (warp >= FL_SOFT && warp < FL_ISSUE) {
        const Converter<HD, BITS, QT> cv(tid - FL_SOFT * 32);
        uint32_t n = 0;
        for (uint32_t s = 0; ok && segment_of(f, s, g); ++s)
#pragma unroll 1
            for (uint32_t t = g.first; t < g.last; ++t, ++n) {
                const uint32_t stage = n % STAGES, slot = n % F::RAWS;
                ok = mbar_wait_warp(b_rfull + 8 * slot, (n / F::RAWS) & 1u, FL_WAIT, s_abort);
                if (!ok) break;
                if (n >= STAGES) ok = mbar_wait_warp(b_free + 8 * stage, (n / STAGES - 1) & 1u, FL_WAIT, s_abort);
                if (!ok) break;
                const uint32_t blocks = reinterpret_cast<volatile uint32_t *>(smem + 528)[slot];
                cv.put(s_raw + slot * F::RAW, s_k + stage * 2 * F::K_TILE, smem + F::CONSTS + stage * (FL_KT / 2) * F::CONST, blocks, p.a.prefix_len - t * FL_KT);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(b_full + 8 * stage);
                    mbar_arrive(b_rfree + 8 * slot);
                }
            }
    } else if (warp == FL_ISSUE) {
        // fp32 accumulators, fp16 operands; A and B K-major for S, B with its columns consecutive for O
        constexpr uint32_t id_s = (1u << 4) | ((FL_KT >> 3) << 17) | ((FLASH_ROWS >> 4) << 24);
        constexpr uint32_t id_o = (1u << 4) | (1u << 16) | (((G == 1 ? HD : 64) >> 3) << 17) | ((FLASH_ROWS >> 4) << 24);
        uint32_t n0 = 0, done[2] = {0, 0};             // tiles of the CTA before the segment; tiles of the streams before it
        for (uint32_t s = 0; ok && segment_of(f, s, g); ++s) {
            const uint32_t n = g.last - g.first, count[2] = {f.halved ? (n + 1) / 2 : n, f.halved ? n / 2 : n};
            auto tile_of = [&](uint32_t st, uint32_t i) { return n0 + (f.halved ? 2 * i + st : i); };
            auto scores = [&](uint32_t st, uint32_t i) {
                const uint32_t tile = tile_of(st, i), stage = tile % STAGES, use = done[st] + i, buf = G == 1 ? use & 1u : 0u;
                if (!mbar_wait_warp(b_full + 8 * stage, (tile / STAGES) & 1u, FL_WAIT, s_abort)) return false;
                tc_fence_after();
                const uint32_t t_s = tmem + st * t_stream + buf * FL_KT;
                const uint64_t q = desc_k(s_q + (f.halved ? 0u : st) * F::Q_TILE), k = desc_k(s_k + stage * 2 * F::K_TILE);          // further operands: addresses in units of 16 bytes
                if (elected()) {
#pragma unroll
                    for (uint32_t c = 0; c < HD / 16; ++c)
#pragma unroll
                        for (uint32_t x = 0; x < QT; ++x)
                            mma_ss(t_s + (G == 2 ? c / 4 * FL_KT : 0u), q + ((x * F::Q_TILE + (c / 4) * FLASH_ROWS * 128 + (c % 4) * 32) >> 4), k + (((c / 4) * FL_KT * 128 + (c % 4) * 32) >> 4), id_s,
                                   (x == 0 && (G == 2 ? c % 4 : c) == 0) ? 0u : 1u);
                    tc_commit(b_s + 8 * (2 * st + buf));
                }
                __syncwarp();
                return true;
            };
            ok = mbar_wait_warp(b_q, s & 1u, FL_WAIT, s_abort);
            for (uint32_t st = 0; ok && st < 2; ++st)
                if (count[st] > 0) ok = scores(st, 0);
            for (uint32_t i = 0; ok && i < count[0]; ++i) {
                auto next_scores = [&](uint32_t st) {
                    if (G != 1 || i + 1 >= count[st]) return true;
                    // the weights of tile i - 1 lie where S of tile i + 1 goes
                    if (i >= 1 && !mbar_wait_warp(b_o + 8 * st, (done[st] + i - 1) & 1u, FL_WAIT, s_abort)) return false;
                    return scores(st, i + 1);
                };
                // Both next scores ahead of either's values, since a stream that waits for the other's weights here holds both back.  Streams over
                // the same tiles use tiles i and i + 1 then, streams of even and odd tiles 2 i .. 2 i + 3: with three stages these go one after
                // the other (2 i .. 2 i + 2), or they would wait for ever for the fourth.
                const bool both = !f.halved || STAGES >= 4;
                for (uint32_t st = 0; ok && both && st < 2; ++st) ok = next_scores(st);
                for (uint32_t st = 0; ok && st < 2; ++st) {
                    if (i >= count[st]) continue;
                    if (!both) ok = next_scores(st);
                    if (!ok) break;
                    const uint32_t use = done[st] + i, buf = G == 1 ? use & 1u : 0u, tile = tile_of(st, i), stage = tile % STAGES;
                    ok = mbar_wait_warp(b_p + 8 * (2 * st + buf), (G == 1 ? use >> 1 : use) & 1u, FL_WAIT, s_abort);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t t_p = tmem + st * t_stream + buf * FL_KT, t_o = tmem + st * t_stream + 128;
                    const uint64_t v = desc_mn(s_k + stage * 2 * F::K_TILE + F::K_TILE, FL_KT * 128);
                    if (elected()) {
#pragma unroll
                        for (uint32_t x = 0; x < G; ++x)
#pragma unroll
                            for (uint32_t y = 0; y < PT; ++y)
#pragma unroll
                                for (uint32_t k = 0; k < FL_KT / 16; ++k)
                                    mma_ts(t_o + x * 64, t_p + (x * PT + y) * 32 + k * 8, v + ((x * FL_KT * 128 + k * 16 * 128) >> 4), id_o, (i | y | k) != 0 ? 1u : 0u);
                        if (f.halved || st == 1) tc_commit(b_free + 8 * stage);
                        tc_commit(b_o + 8 * st);
                    }
                    __syncwarp();
                }
                if (G == 2)
                    for (uint32_t st = 0; ok && st < 2; ++st)
                        if (i + 1 < count[st]) {
                            ok = mbar_wait_warp(b_o + 8 * st, (done[st] + i) & 1u, FL_WAIT, s_abort);
                            if (!ok) break;
                            ok = scores(st, i + 1);
                        }
            }
            if (elected()) tc_commit(b_end);
            __syncwarp();
            n0 += n;
            done[0] += count[0];
            done[1] += count[1];
        }
        if (elected()) tc_commit(b_last);               // also after a wait that gave up: the products in flight end before the CTA leaves
        for (uint32_t spin = 0; spin < FL_WAIT && !mbar_try_wait(b_last, 0); ++spin) {}
        if (!ok && lane == 0) atomicCAS(p.a.pool.err, 0u, 1u);
    } else {
        const uint32_t st = warp / 4, quarter = warp % 4, lr = lane >> 2, lc = lane & 3u;
        const uint32_t group = p.a.heads / p.a.pool.d.kv_heads, all = p.a.n_tok * group;
        const uint32_t t_s0 = tmem + st * t_stream + ((quarter * 32u) << 16), t_o = t_s0 + 128;
        uint32_t n0 = 0, done = 0;
        for (uint32_t s = 0; ok && segment_of(f, s, g); ++s) {
            if (tid == 0) {                            // the products that read the last segment's queries have ended (b_end)
                const uint32_t bytes = (f.halved ? QT : 2) * F::Q_TILE;
                mbar_expect_tx(b_q, bytes);
                for (uint32_t i = 0; i < bytes; i += F::Q_TILE) bulk_g2s(s_q + i, f.queries + (size_t)g.item * bytes + i, F::Q_TILE, b_q);
            }
            const uint32_t n = g.last - g.first, count = f.halved ? (n + 1 - st) / 2 : n;
            const uint32_t r0 = g.item % f.row_tiles * (f.halved ? 1 : 2) * FLASH_ROWS + (f.halved ? 0u : st * FLASH_ROWS), left = all > r0 ? all - r0 : 0;          // rows of the stream's tile
            const bool idle = quarter * 32 >= left;
            float c[4], m[4], l[4];                // rows quarter * 32 + lr + 8 k
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                c[k] = __ldcg(f.factors + g.item * (f.halved ? 1 : 2) * FLASH_ROWS + (f.halved ? 0u : st * FLASH_ROWS) + quarter * 32 + lr + 8 * k);
                m[k] = -INFINITY;
                l[k] = 0.0f;
            }
            for (uint32_t i = 0; i < count; ++i) {
                const uint32_t use = done + i, buf = G == 1 ? use & 1u : 0u, tile = n0 + (f.halved ? 2 * i + st : i), stage = tile % STAGES;
                ok = mbar_wait_warp(b_s + 8 * (2 * st + buf), (G == 1 ? use >> 1 : use) & 1u, FL_WAIT, s_abort);
                if (!ok) break;
                ok = mbar_wait_warp(b_full + 8 * stage, (tile / STAGES) & 1u, FL_WAIT, s_abort);          // this thread's view of the constants
                if (!ok) break;
                tc_fence_after();
                const uint32_t s_const = sbase + F::CONSTS + stage * (FL_KT / 2) * F::CONST;
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half) {
                    if (idle) break;
                    const uint32_t t_s = t_s0 + buf * FL_KT + ((16u * half) << 16);
                    uint32_t v[G * 32];
                    tm_ld_frag64(t_s, v);
                    if (G == 2) tm_ld_frag64(t_s + FL_KT, v + (G - 1) * 32);
                    tm_ld_wait();
                    u64 x[8][2];
                    const u64 ca = pair_of(c[2 * half], c[2 * half]), cb = pair_of(c[2 * half + 1], c[2 * half + 1]);
                    float ta = -INFINITY, tb = -INFINITY;
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k) {
                        const uint32_t j = 4 * k + lc;          // pair of columns
                        u64 ks, lv;
                        if (G == 1) {
                            lds_pairs(s_const + j * 16, ks, lv);
                            x[k][0] = fma2(mul2(pair_of(v[4 * k], v[4 * k + 1]), ca), ks, lv);
                            x[k][1] = fma2(mul2(pair_of(v[4 * k + 2], v[4 * k + 3]), cb), ks, lv);
                        } else {
                            u64 k2;
                            lds_pairs(s_const + j * 48, ks, k2);
                            lv = lds_pair(s_const + j * 48 + 16);
                            constexpr uint32_t H = (G - 1) * 32;
                            x[k][0] = fma2(fma2(pair_of(v[H + 4 * k], v[H + 4 * k + 1]), k2, mul2(pair_of(v[4 * k], v[4 * k + 1]), ks)), ca, lv);
                            x[k][1] = fma2(fma2(pair_of(v[H + 4 * k + 2], v[H + 4 * k + 3]), k2, mul2(pair_of(v[4 * k + 2], v[4 * k + 3]), ks)), cb, lv);
                        }
                        float lo, hi;
                        unpair(x[k][0], lo, hi);
                        ta = max3(ta, lo, hi);
                        unpair(x[k][1], lo, hi);
                        tb = max3(tb, lo, hi);
                    }
                    if (__any_sync(0xffffffffu, ta > m[2 * half] + MAX_ROOM || tb > m[2 * half + 1] + MAX_ROOM)) {
#pragma unroll
                        for (uint32_t o = 1; o < 4; o <<= 1) {
                            ta = fmaxf(ta, __shfl_xor_sync(0xffffffffu, ta, o));
                            tb = fmaxf(tb, __shfl_xor_sync(0xffffffffu, tb, o));
                        }
                        const float ma = fmaxf(m[2 * half], ta - MAX_BELOW), mb = fmaxf(m[2 * half + 1], tb - MAX_BELOW);
                        if (i > 0) {
                            ok = mbar_wait_warp(b_o + 8 * st, (use - 1) & 1u, FL_WAIT, s_abort);
                            if (!ok) break;
                            tc_fence_after();
                            const float aa = ma == -INFINITY ? 1.0f : exp2_approx(m[2 * half] - ma), ab = mb == -INFINITY ? 1.0f : exp2_approx(m[2 * half + 1] - mb);
#pragma unroll 1
                            for (uint32_t col = 0; col < HD; col += 32) {
                                uint32_t o[16];
                                tm_ld_frag32(t_o + ((16u * half) << 16) + col, o);
                                tm_ld_wait();
#pragma unroll
                                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * ((k & 2) ? ab : aa));
                                tm_st_frag32(t_o + ((16u * half) << 16) + col, o);
                            }
                            l[2 * half] *= aa;
                            l[2 * half + 1] *= ab;
                        }
                        m[2 * half] = ma;
                        m[2 * half + 1] = mb;
                    }
                    const float na = m[2 * half] == -INFINITY ? 0.0f : -m[2 * half], nb = m[2 * half + 1] == -INFINITY ? 0.0f : -m[2 * half + 1];
                    const u64 ma = pair_of(na, na), mb = pair_of(nb, nb);
                    u64 sa = 0, sb = 0;
                    uint32_t w[G][PT][16];
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k) {
                        const uint32_t j = 4 * k + lc;
                        u64 iv, pa = 0, pb = 0;
                        if (G == 1) {
                            iv = lds_pair(s_const + FL_KT / 2 * 16 + j * 8);
                        } else {
                            iv = lds_pair(s_const + j * 48 + 24);
                            lds_pairs(s_const + j * 48 + 32, pa, pb);
                        }
#pragma unroll
                        for (uint32_t r = 0; r < 2; ++r) {
                            float lo, hi;
                            unpair(add2(x[k][r], r == 0 ? ma : mb), lo, hi);
                            lo = exp2_approx(lo);
                            hi = exp2_approx(hi);
                            const u64 e = pair_of(lo, hi);
                            if (r == 0) sa = fma2(e, iv, sa);
                            else sb = fma2(e, iv, sb);
#pragma unroll
                            for (uint32_t y = 0; y < G; ++y) {
                                if (G == 2) unpair(mul2(e, y == 0 ? pa : pb), lo, hi);
                                w[y][0][2 * k + r] = half2_bits(lo, hi);
                                if (PT == 2) {
                                    const float2 t = __half22float2(*reinterpret_cast<const __half2 *>(&w[y][0][2 * k + r]));
                                    w[y][PT - 1][2 * k + r] = half2_bits(lo - t.x, hi - t.y);
                                }
                            }
                        }
                    }
                    float lo, hi;
                    unpair(sa, lo, hi);
                    l[2 * half] += lo + hi;
                    unpair(sb, lo, hi);
                    l[2 * half + 1] += lo + hi;
#pragma unroll
                    for (uint32_t y = 0; y < G; ++y)
#pragma unroll
                        for (uint32_t z = 0; z < PT; ++z) tm_st_words32(t_s + (y * PT + z) * 32, w[y][z]);
                }
                if (!ok) break;
                tm_st_wait();
                tc_fence_before();
                mbar_arrive(b_p + 8 * (2 * st + buf));
            }
            if (!ok) break;
            // the segment's last update by a barrier of its own: the phases of b_o may be two behind here, and a parity tells only neighbours apart
            ok = mbar_wait_warp(b_end, s & 1u, FL_WAIT, s_abort);
            if (!ok) break;
            tc_fence_after();
            float *slot = p.near + (size_t)(blockIdx.x + g.item) * flash_slot_floats(HD) + st * flash_slot_floats(HD) / 2;
            if (!idle) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (uint32_t o = 1; o < 4; o <<= 1) l[k] += __shfl_xor_sync(0xffffffffu, l[k], o);
#pragma unroll 1
                for (uint32_t half = 0; half < 2; ++half)
#pragma unroll 1
                    for (uint32_t col = 0; col < HD; col += 32) {
                        uint32_t o[16];
                        tm_ld_frag32(t_o + ((16u * half) << 16) + col, o);
                        tm_ld_wait();
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k) {          // row k & 1, columns of group k / 2
                            const uint32_t row = quarter * 32 + half * 16 + lr + 8 * (k & 1u);
                            const float2 val = count == 0 ? make_float2(0.0f, 0.0f) : make_float2(__uint_as_float(o[4 * (k / 2) + 2 * (k & 1u)]), __uint_as_float(o[4 * (k / 2) + 2 * (k & 1u) + 1]));
                            if (row < left) *reinterpret_cast<float2 *>(slot + row * HD + col + 8 * (k / 2) + 2 * lc) = val;
                        }
                    }
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    const uint32_t row = quarter * 32 + lr + 8 * k;
                    if (lc == 0 && row < left) *reinterpret_cast<float2 *>(slot + FLASH_ROWS * HD + 2 * row) = make_float2(m[k], l[k]);
                }
            }
            tc_fence_before();
            n0 += n;
            done += count;
        }
        if (!ok && lane == 0) atomicCAS(p.a.pool.err, 0u, 1u);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == FL_ISSUE) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(FL_COLS) : "memory");
    }
}

template <int HD, int BITS, int QT, int PT> cudaError_t flash_go(cudaStream_t s, const SplitArgs &p) {
    constexpr uint32_t smem = Flash<HD, BITS, QT>::SMEM;
    static_assert(smem <= 232448, "shared memory of an SM");
    const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void *>(pool_flash_kernel<HD, BITS, QT, PT>), smem);
    if (e != cudaSuccess) return e;
    const uint32_t line = p.flash.items * p.flash.tiles, rows = p.flash.items * (p.flash.halved ? 1 : 2) * FLASH_ROWS;
    const cudaError_t q = launch_kernel(pool_query_kernel<HD, QT>, dim3(rows * (HD / 8) / QK_THREADS), dim3(QK_THREADS), 0, s, true, p);
    if (q != cudaSuccess) return q;
    return launch_kernel(pool_flash_kernel<HD, BITS, QT, PT>, dim3((line - 1) / p.flash.part + 1), dim3(FL_THREADS), smem, s, true, p);
}
template <int HD, int BITS> cudaError_t flash_type(cudaStream_t s, const SplitArgs &p) {
    const uint32_t type = p.a.q.type;
    return type == TYPE_F32 ? flash_go<HD, BITS, 2, 2>(s, p) : type == TYPE_F16 ? flash_go<HD, BITS, 2, 1>(s, p) : flash_go<HD, BITS, 1, 1>(s, p);
}

}  // namespace

cudaError_t launch_pool_flash(cudaStream_t s, const SplitArgs &p) {
    const PoolShape &d = p.a.pool.d;
    return d.head_dim == 128 ? (d.bits == 8 ? flash_type<128, 8>(s, p) : flash_type<128, 4>(s, p)) : d.bits == 8 ? flash_type<64, 8>(s, p) : flash_type<64, 4>(s, p);
}

}  // namespace k2t
