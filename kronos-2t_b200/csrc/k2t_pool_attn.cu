// Attention over the pool for few query rows at a time: tables of pages, chosen pages, and a shared prefix with up to a tile of rows.
//   score t_ij = (c_i q_i . code_j) ks_j, kept as x_ij = t_ij + log2 vs_j, so that 2^x is the weight already times the value's scale and
//   every operand of a product is a code (whole numbers up to 127, exact halves) or a weight of at most 2^15;
//   numerator O_i = sum_j 2^(x_ij - m_i) codev_j, denominator l_i = sum_j 2^(x_ij - m_i) / vs_j, with the running maximum m_i of x.
// Rows of zeros have vs = 2^-64 (see weight_scale): with 1 they took the digits of the others' weights, which are all of the output.
// Positions out of sight have ks = 0, log2 vs = -inf, 1 / vs = 0: no mask per element, and nothing of theirs is multiplied.
//
// A CTA works with 8 or 16 query rows (queries of one kv head, so a cached row is read once for the heads that share it).  Its four warps
// take every fourth block of 16 positions, which bulk copies bring into a ring of each warp's own, and join their results at the end of an item.  Positions are the ROWS of the products
// (m16n8k16, halves): S^T = K Q^T, O^T = V^T P^T, so eight queries cost one tile where queries as rows would pad them to sixteen; scores,
// exponentials and accumulators halve with them.  What is left is the expansion of codes to halves, 2.25 instructions a value pair.
// Items (token, kv head) are cut into equal pieces, one per CTA, or, where there are more of them than CTAs and they are long, their blocks are one
// line cut into equal parts, so that ragged lengths keep every CTA busy to the end (own_pieces).  An item that lies in one part is finished
// there; the others leave partial results, which pool_merge_kernel joins.
#include <algorithm>

#include "k2t_flash_tc.cuh"
#include "k2t_kv_pool.cuh"
#include "k2t_pool_attn.h"

namespace k2t {
namespace {

constexpr uint32_t SP_WARPS = 4, SP_STAGES = 2, WAIT_LIMIT = 1u << 22;
// CTAs on an SM, by the registers of a kernel that spills nothing worth naming
constexpr uint32_t split_ctas(uint32_t hd, uint32_t bits, bool two_terms, bool two_weights, uint32_t nr) {
    if (hd == 64) return nr == 1 ? 4 : 3;
    if (nr == 2) return two_terms || bits == 4 ? 2 : 3;
    return 4 - (two_weights ? 1 : 0) - (two_terms && bits == 4 ? 1 : 0);
}
// Shared memory: the warps' rings, the queries as halves, and the warps' results of eight rows (rows HD + 4 floats apart, so that lanes of
// neighbouring rows meet in other banks).
template <int HD, int BITS, int QT, int NR> struct SplitSmem {
    static constexpr uint32_t PITCH = HD + 4, QUERY = SP_WARPS * SP_STAGES * PoolBlock<HD, BITS>::BYTES, JOIN = QUERY + NR * QT * 8 * HD * 2,
                              ML = JOIN + SP_WARPS * 8 * PITCH * 4, FACTOR = ML + SP_WARPS * 8 * 8, BYTES = FACTOR + NR * 8 * 4;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {       // 8 x 8 halves over the warp
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <int WORDS> __device__ __forceinline__ void lds_words(uint32_t addr, uint32_t *w) {
    if constexpr (WORDS == 4) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
    else if constexpr (WORDS == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}
__device__ __forceinline__ float lds_f32(uint32_t addr) { float v; asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr)); return v; }

// The sequence of a token and the rows of it that the token sees, cut to what its table holds.
__device__ __forceinline__ uint32_t seen_rows(const PoolAttnArgs &a, uint32_t t, int32_t &seq) {
    seq = a.seq != nullptr ? __ldcg(a.seq + t) : (int32_t)t;
    const int32_t len = seq < 0 ? 0 : __ldcg(a.lens + t);
    const uint64_t room = (uint64_t)a.pages_stride << a.pool.d.page_shift;
    if (len <= 0) return 0;
    if ((uint64_t)len > room) { pool_bad_page(a.pool); return (uint32_t)room; }
    return (uint32_t)len;
}
__device__ __forceinline__ uint32_t item_blocks(const SplitArgs &p, uint32_t t) {       // of one (token, kv head, tile of rows)
    if (p.a.chosen != nullptr) return p.a.top << (p.a.pool.d.page_shift - 4);
    int32_t seq;
    return (seen_rows(p.a, t, seq) + POOL_ROWS - 1) / POOL_ROWS;
}

// One item of the line and the block of it that is next.
struct Item {
    uint32_t index, t, h, rb;          // of the prefix items: (h, rb)
    uint32_t next, blocks, len;        // positions in sight: len
    const int32_t *list;               // pages, or choices among the pages of `table`
    const int32_t *table;
    bool prefix;
};

__device__ __forceinline__ void item_fill(const SplitArgs &p, Item &it) {
    if (it.prefix) {
        it.list = p.a.prefix_pages;
        it.len = p.a.prefix_len;
        it.blocks = prefix_blocks(p);
        return;
    }
    int32_t seq;
    it.len = seen_rows(p.a, it.t, seq);
    it.table = p.a.pages + (size_t)max(seq, 0) * p.a.pages_stride;
    const bool chosen = p.a.chosen != nullptr;
    it.list = chosen ? p.a.chosen + ((size_t)it.t * p.a.pool.d.kv_heads + it.h) * p.a.top : it.table;
    it.blocks = chosen ? p.a.top << (p.a.pool.d.page_shift - 4) : (it.len + POOL_ROWS - 1) / POOL_ROWS;
}

// Sums of the tokens' blocks over a warp: the whole, and the place of the token that holds block `x` of them (counted per kv head and tile).
__device__ __forceinline__ uint64_t warp_total(const SplitArgs &p, uint32_t lane) {
    uint64_t sum = 0;
#pragma unroll 4
    for (uint32_t t = lane; t < p.a.n_tok; t += 32) sum += item_blocks(p, t);
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    return sum;
}
__device__ __forceinline__ void warp_find(const SplitArgs &p, uint64_t x, uint32_t lane, uint32_t &t, uint64_t &before, uint32_t &blocks) {
    uint64_t base = 0;
#pragma unroll 1
    for (uint32_t t0 = 0; t0 < p.a.n_tok; t0 += 32) {
        const uint32_t n = t0 + lane < p.a.n_tok ? item_blocks(p, t0 + lane) : 0;
        uint64_t upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const uint64_t y = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= (uint32_t)o) upto += y; }
        const uint32_t hit = __ballot_sync(0xffffffffu, base + upto > x);
        if (hit != 0) {
            const uint32_t l = __ffs(hit) - 1;
            t = t0 + l;
            blocks = __shfl_sync(0xffffffffu, n, l);
            before = base + __shfl_sync(0xffffffffu, upto, l) - blocks;
            return;
        }
        base += __shfl_sync(0xffffffffu, upto, 31);
    }
    t = p.a.n_tok; before = base; blocks = 1;            // not reached: x lies below the total
}

// The item that holds block x of the line: tokens in order, of a token its kv heads, of those their tiles.
__device__ __forceinline__ void item_at(const SplitArgs &p, uint64_t x, uint32_t lane, Item &it) {
    const uint32_t per = p.a.pool.d.kv_heads * p.rbo;
    uint32_t blocks;
    uint64_t before;
    warp_find(p, x / per, lane, it.t, before, blocks);
    const uint64_t in = x - before * per;
    const uint32_t sub = (uint32_t)(in / blocks);
    it.prefix = false;
    it.h = sub / p.rbo;
    it.rb = sub % p.rbo;
    it.index = it.t * per + sub;
    it.next = (uint32_t)(in - (uint64_t)sub * blocks);
    item_fill(p, it);
}
// The item behind this one; tokens without a block are passed over (the caller knows that there is one).
__device__ __forceinline__ bool item_after(const SplitArgs &p, Item &it) {          // of a line; whether its list is another one
    it.next = 0;
    it.index += 1;
    if (++it.rb == p.rbo) { it.rb = 0; it.h += 1; }
    if (it.h < p.a.pool.d.kv_heads) return false;
    it.h = 0;
    it.t += 1;
    if (it.t < p.a.n_tok) item_fill(p, it);
    while (it.blocks == 0 && it.t + 1 < p.a.n_tok) {
        it.t += 1;
        it.index += p.a.pool.d.kv_heads * p.rbo;
        item_fill(p, it);
    }
    return true;
}

// ------------------------------------------------------------------------------------------------ the warp's rows
// Query row i of an item: whether it exists, its token and head.
__device__ __forceinline__ bool item_row(const SplitArgs &p, const Item &it, uint32_t i, uint32_t &t, uint32_t &head) {
    const uint32_t group = p.a.heads / p.a.pool.d.kv_heads, r = it.rb * p.tile + i;
    t = it.prefix ? r / group : it.t;
    head = it.h * group + (it.prefix ? r % group : r);
    return it.prefix ? t < p.a.n_tok : r < group;
}

// The tile's rows, HD / 8 lanes each, to shared memory: [row][term][element], the 16-byte chunks of a row turned by its number; and their factors.
template <int HD, int QT, int NR> __device__ __forceinline__ void put_queries(const SplitArgs &p, const Item &it, uint32_t tid, uint8_t *s_query, float *s_factor) {
    constexpr uint32_t LANES = HD / 8;
    const uint32_t lane = tid & 31u, l = tid % LANES;
#pragma unroll
    for (uint32_t row0 = 0; row0 < 8 * NR; row0 += SP_WARPS * 32 / LANES) {
        const uint32_t row = row0 + tid / LANES;
        if (row0 + (tid & ~31u) / LANES >= 8 * NR) break;          // whole warps
        uint32_t t, head, hi[4], lo[4];
        const bool there = item_row(p, it, row, t, head);
        const float down = query_halves<HD>(p.a.pool, p.a.q, there, t * p.a.q.token_stride + head * p.a.q.head_stride, l, lane, hi, lo);
        if (l == 0) s_factor[row] = p.a.scale * LOG2E * down;
        uint4 *to = reinterpret_cast<uint4 *>(s_query + row * QT * HD * 2) + (l ^ (row & 7u));
        to[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (QT == 2) to[HD / 8] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}
// Lane (n, t) = (lane / 4, lane % 4) takes of query row n (and n + 8) the elements [16 t, 16 t + 16) of each 64 as its columns of the second
// operand: step i of a group of 64 is elements 4 i .. 4 i + 3 of every lane.  c: factor of the scores of rows 2 t, 2 t + 1.
template <int HD, int QT, int NR> struct Query {
    uint32_t b[NR][QT][HD / 16][2];
    float c[NR][2];
};
template <int HD, int QT, int NR> __device__ __forceinline__ void get_queries(uint32_t s_query, uint32_t s_factor, uint32_t lane, Query<HD, QT, NR> &q) {
    const uint32_t n = lane >> 2, t4 = lane & 3u;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        q.c[r][0] = lds_f32(s_factor + (8 * r + 2 * t4) * 4);
        q.c[r][1] = lds_f32(s_factor + (8 * r + 2 * t4 + 1) * 4);
#pragma unroll
        for (int k = 0; k < QT; ++k)
#pragma unroll
            for (int g = 0; g < HD / 64; ++g)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    uint32_t w[4];
                    lds_words<4>(s_query + ((n + 8 * r) * QT + k) * HD * 2 + (((g * 8 + t4 * 2 + x) ^ n) << 4), w);
                    q.b[r][k][4 * g + 2 * x][0] = w[0]; q.b[r][k][4 * g + 2 * x][1] = w[1];
                    q.b[r][k][4 * g + 2 * x + 1][0] = w[2]; q.b[r][k][4 * g + 2 * x + 1][1] = w[3];
                }
    }
}

// o[r][j]: elements n HD / 8 + 2 j and the next (two groups of 64: n 8 + 2 j of the first, for j >= 4 of the second), of query rows 8 r + 2 t and
// the next; m, l of those rows (l of the lane's positions)
template <int HD, int NR> struct State {
    float o[NR][HD / 16][4], m[NR][2], l[NR][2];
};

// Where a lane's rows lie in a block: row_place of its rows, of which the second pair of keys and of values lies a fixed distance behind the
// first (rows of 32 bytes: values by exclusive-or of the row).
template <int HD, int BITS> struct LanePlaces {
    using B = PoolBlock<HD, BITS>;
    static constexpr uint32_t RB = B::RB;
    uint32_t k[2], v[2];
    __device__ __forceinline__ explicit LanePlaces(uint32_t lane) {
        const uint32_t n = lane >> 2, t = lane & 3u, p0 = 4 * (n >> 1) + (n & 1u);
        k[0] = row_place<RB>(p0, t * (BITS == 8 ? 16 : 8));
        k[1] = RB == 32 || HD == 64 ? row_place<RB>(p0 + 2, t * (BITS == 8 ? 16 : 8)) : row_place<RB>(p0, RB / 2 + t * (BITS == 8 ? 16 : 8));
        v[0] = B::V_AT + row_place<RB>(4 * t, n * (RB / 8 / B::G));
        v[1] = B::V_AT + row_place<RB>(4 * t + 1, n * (RB / 8 / B::G));
    }
    __device__ __forceinline__ uint32_t key(uint32_t at, int j, int g) const { return HD == 64 ? at + k[j] : at + k[g] + j * 2 * RB; }          // row p0 + 2 j, group g
    // row 4 t + i; the second group of 64 elements of a 4-bit row lies 32 bytes on, where no exclusive-or of the first reaches but its own
    __device__ __forceinline__ uint32_t value2(uint32_t at, int i) const { return at + (v[i & 1] ^ 32u) + (i >> 1) * 2 * RB; }
    __device__ __forceinline__ uint32_t value(uint32_t at, int i) const { return RB == 32 ? at + (v[0] ^ (i * 32)) : at + v[i & 1] + (i >> 1) * 2 * RB; }          // row 4 t + i
};

// One block of 16 positions, `valid` of them in sight, at shared address `at`.
template <int HD, int BITS, int QT, int PT, int NR>
__device__ __forceinline__ void block_step(uint32_t at, uint32_t valid, uint32_t lane, const LanePlaces<HD, BITS> &place, const Expand &ex, const Query<HD, QT, NR> &q, State<HD, NR> &st) {
    using B = PoolBlock<HD, BITS>;
    constexpr int G = B::G;
    const uint32_t n = lane >> 2;
    // Row i of the products is position 4 (i / 2) + i % 2 for the first eight, two further for the others: the lane has rows n and n + 8.
    const uint32_t p0 = 4 * (n >> 1) + (n & 1u);
    float s[NR][G][4];                     // rows n, n + 8 of queries 2 t, 2 t + 1, of each group of 64 elements that has a scale
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int g = 0; g < G; ++g) s[r][g][0] = s[r][g][1] = s[r][g][2] = s[r][g][3] = 0.0f;
    uint32_t kw[HD / 64][2][4];
#pragma unroll
    for (int g = 0; g < HD / 64; ++g)
#pragma unroll
        for (int j = 0; j < 2; ++j) lds_words<BITS == 8 ? 4 : 2>(place.key(at, j, g), kw[g][j]);
    uint32_t sc[2][2];                         // scales as they lie: keys, values of p0, p0 + 2
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t off = BITS == 4 && G == 1 ? (p0 & ~1u) * 2 + 4 * j : p0 * 4 + 8 * j;          // of one group of 4 bits two positions share a word
        lds_words<1>(at + B::KS_AT + off, &sc[0][j]);
        lds_words<1>(at + B::VS_AT + off, &sc[1][j]);
    }
#pragma unroll
    for (int g = 0; g < HD / 64; ++g) {
        uint32_t w[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (BITS == 8) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[j][i] = kw[g][j][i];
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) { w[j][2 * i] = ex.centroids4(kw[g][j][i]); w[j][2 * i + 1] = ex.centroids4(kw[g][j][i] >> 16); }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t a[4] = {ex.halves_lo(w[0][i]), ex.halves_lo(w[1][i]), ex.halves_hi(w[0][i]), ex.halves_hi(w[1][i])};
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
                for (int k = 0; k < QT; ++k) mma_f16(s[r][G == 1 ? 0 : g], a, q.b[r][k][4 * g + i][0], q.b[r][k][4 * g + i][1]);
        }
    }
    // values of positions 4 t .. 4 t + 3, asked for ahead of the softmax
    constexpr int W = HD / 32, VW = BITS == 8 ? W : W / 2;          // words of four elements; as they lie
    uint32_t vw[4][VW];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lds_words<VW / G>(place.value(at, i), vw[i]);
        if (G == 2) lds_words<VW / G>(place.value2(at, i), vw[i] + VW / 2);
    }
    // constants of positions p0 and p0 + 2
    float ks[G][2], lv[2], iv[2], part[G][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t pos = p0 + 2 * j;
        float v[G], top;
        if (BITS == 8) {
            ks[0][j] = __uint_as_float(sc[0][j]);
            v[0] = __uint_as_float(sc[1][j]);
        } else if (G == 2) {
            ks[0][j] = __uint_as_float(sc[0][j] << 16); ks[G - 1][j] = __uint_as_float(sc[0][j] & 0xFFFF0000u);
            v[0] = __uint_as_float(sc[1][j] << 16); v[G - 1] = __uint_as_float(sc[1][j] & 0xFFFF0000u);
        } else {
            ks[0][j] = __uint_as_float(pos & 1u ? sc[0][j] & 0xFFFF0000u : sc[0][j] << 16);
            v[0] = __uint_as_float(pos & 1u ? sc[1][j] & 0xFFFF0000u : sc[1][j] << 16);
        }
        // scales are not negative, and all groups of a row are NaN or none; of a row of zeros 8-bit codes are 0, groups of 4 bits have a factor
        top = weight_scale(G == 1 ? v[0] : fmaxf(v[0], v[G - 1]));
        if (pos < valid) {
            lv[j] = log2_approx(top);
            iv[j] = rcp_approx(top);
#pragma unroll
            for (int g = 0; g < G; ++g) part[g][j] = v[g] * iv[j];
        } else {
            lv[j] = -INFINITY;
            iv[j] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g) ks[g][j] = part[g][j] = 0.0f;
        }
    }
    float x[NR][4], top[NR][2];                // [position p0 | p0 + 2][query 2 t | 2 t + 1]
    bool grows = false;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float d = s[r][0][e] * ks[0][e >> 1];
            if (G == 2) d = __fmaf_rn(s[r][G - 1][e], ks[G - 1][e >> 1], d);
            x[r][e] = __fmaf_rn(d, q.c[r][e & 1], lv[e >> 1]);
        }
        top[r][0] = fmaxf(x[r][0], x[r][2]);
        top[r][1] = fmaxf(x[r][1], x[r][3]);
        grows |= top[r][0] > st.m[r][0] + MAX_ROOM || top[r][1] > st.m[r][1] + MAX_ROOM;
    }
    // weights stay within halves, sums are exact in either case
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float y = top[r][e];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, o));
                const float m = fmaxf(st.m[r][e], y - MAX_BELOW), al = m == -INFINITY ? 1.0f : exp2_approx(st.m[r][e] - m);
                st.m[r][e] = m;
                st.l[r][e] *= al;
#pragma unroll
                for (int j = 0; j < HD / 16; ++j) { st.o[r][j][e] *= al; st.o[r][j][2 + e] *= al; }
            }
    }
    uint32_t b[NR][G][PT][2];                  // weights as the second operand: transposed, the lane's positions are 4 t .. 4 t + 3 of query n
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const float base0 = st.m[r][0] == -INFINITY ? 0.0f : st.m[r][0], base1 = st.m[r][1] == -INFINITY ? 0.0f : st.m[r][1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[r][e] = exp2_approx(x[r][e] - (e & 1 ? base1 : base0));
            st.l[r][e & 1] = __fmaf_rn(x[r][e], iv[e >> 1], st.l[r][e & 1]);
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float u = BITS == 4 ? x[r][2 * j] * part[g][j] : x[r][2 * j], v = BITS == 4 ? x[r][2 * j + 1] * part[g][j] : x[r][2 * j + 1];
                const uint32_t hi = half2_bits(u, v);
                b[r][g][0][j] = transposed(hi);
                if constexpr (PT == 2) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                    b[r][g][PT - 1][j] = transposed(half2_bits(u - f.x, v - f.y));
                }
            }
    }
    // values: columns of the first operand are positions, two of them a word; rows n and n + 8 of tile j are the elements of o[.][j]
    uint32_t v[4][W];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < VW; ++k) {
            if (BITS == 8) {
                v[i][k] = vw[i][k];
            } else {
                v[i][2 * k] = ex.centroids4(vw[i][k]);
                v[i][2 * k + 1] = ex.centroids4(vw[i][k] >> 16);
            }
        }
#pragma unroll
    for (int k = 0; k < W; ++k) {
        const uint32_t lo01 = prmt(v[0][k], v[1][k], 0x5140u), lo23 = prmt(v[2][k], v[3][k], 0x5140u), hi01 = prmt(v[0][k], v[1][k], 0x7362u), hi23 = prmt(v[2][k], v[3][k], 0x7362u);
        const uint32_t first[4] = {ex.halves_lo(lo01), ex.halves_hi(lo01), ex.halves_lo(lo23), ex.halves_hi(lo23)}, second[4] = {ex.halves_lo(hi01), ex.halves_hi(hi01), ex.halves_lo(hi23), ex.halves_hi(hi23)};
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
                for (int y = 0; y < PT; ++y) mma_f16(st.o[r][2 * k + e], e == 0 ? first : second, b[r][G == 1 ? 0 : k / (W / 2)][y][0], b[r][G == 1 ? 0 : k / (W / 2)][y][1]);
    }
}

template <int HD, int BITS, int QT, int PT, int NR>
__global__ void __launch_bounds__(SP_WARPS * 32, split_ctas(HD, BITS, QT == 2, PT == 2, NR)) pool_split_kernel(const __grid_constant__ SplitArgs p) {
    using B = PoolBlock<HD, BITS>;
    using S = SplitSmem<HD, BITS, QT, NR>;
    extern __shared__ __align__(128) uint8_t smb[];
    __shared__ __align__(8) uint64_t bars[SP_WARPS][SP_STAGES];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t sbase = (uint32_t)__cvta_generic_to_shared(smb), ring = sbase + warp * SP_STAGES * B::BYTES, bar = (uint32_t)__cvta_generic_to_shared(bars[warp]);
    const PoolShape &d = p.a.pool.d;
    const uint32_t bs = d.page_shift - 4, in_page = (1u << bs) - 1u;
    const bool listed = p.a.chosen == nullptr;
    if (lane == 0) {
        for (uint32_t i = 0; i < SP_STAGES; ++i) mbar_init(bar + 8 * i, 1);
        fence_mbar_init();
    }
    __syncwarp();
    // Behind the prefix's kernel: that one started its dependents when everything it reads was there, and writes nothing that is read here, so
    // only the end of this kernel waits for it -- for the merge, which waits for this one alone.
    const bool behind = p.flash.on;
    if (!behind) {
        pdl_wait();
        pdl_trigger();
    }
    Item it;
    uint32_t left;                             // blocks of the CTA's part
    const bool near = blockIdx.x < p.near_units;
    const uint32_t unit = near ? blockIdx.x : blockIdx.x - p.near_units, pieces = near ? p.near_pieces : p.pieces;
    if (pieces != 0) {             // the part is a piece of one item, which may hold no block at all
        const uint32_t tiles = near ? p.rbp : p.rbo, per = d.kv_heads * tiles, item = unit / pieces, piece = unit % pieces;
        it.prefix = near;
        it.index = item;
        it.t = item / per;
        it.h = item % per / tiles;
        it.rb = item % tiles;
        item_fill(p, it);
        const uint32_t part = piece_blocks(pieces, it.blocks);
        it.next = min(it.blocks, piece * part);
        left = min(it.blocks - it.next, part);
        if (piece > 0 && left == 0) {          // fewer blocks than pieces; the first one stands for an item without any
            if (behind) pdl_wait();
            return;
        }
    } else {
        const uint64_t all = warp_total(p, lane) * d.kv_heads * p.rbo, part = part_blocks(all, p.units), x = (uint64_t)unit * part;
        if (x >= all) {
            if (behind) pdl_wait();
            return;
        }
        left = (uint32_t)min(part, all - x);
        item_at(p, x, lane, it);
    }
    // What the warp asks for next: block ask.next of an item, every fourth up to ask_end; ask_left blocks of the part lie behind that item.
    Item ask = it;
    uint32_t ask_end = it.next + min(left, it.blocks - it.next), ask_left = left - (ask_end - it.next);
    ask.next += warp;
    uint32_t asked = 0, held = 0, phase = 0;          // a byte per stage: positions in sight; a bit per stage: parity of its next copy
    int32_t page = 0, first = 0;               // over the lanes: 32 pages of the list, and where a chosen one begins (below 0: nothing in sight)
    uint32_t pages_at = ~0u;                   // which 32

    auto request = [&]() {                     // one block, into stage asked % SP_STAGES
        while (ask.next >= ask_end) {
            if (ask_left == 0) return;
            if (item_after(p, ask)) pages_at = ~0u;
            ask_end = min(ask_left, ask.blocks);
            ask_left -= ask_end;
            ask.next = warp;
        }
        const uint32_t b = ask.next, entry = b >> bs;
        if (pages_at != entry >> 5) {
            pages_at = entry >> 5;
            const uint32_t e = (entry & ~31u) + lane, pages = (ask.len + (1u << d.page_shift) - 1) >> d.page_shift;
            page = first = 0;
            if (listed || ask.prefix) {
                if (e < pages) page = __ldcg(ask.list + e);
            } else {
                const int32_t c = e < p.a.top ? __ldcg(ask.list + e) : -1;
                first = c >= 0 && (uint32_t)c < pages ? c : -1;
                if (first >= 0) page = __ldcg(ask.table + c);
            }
            if (page < 0 || (uint32_t)page >= d.num_pages) { pool_bad_page(p.a.pool); page = 0; first = -1; }
        }
        const int32_t pg = __shfl_sync(0xffffffffu, page, entry & 31u), begins = __shfl_sync(0xffffffffu, first, entry & 31u);
        const uint32_t pos = listed || ask.prefix ? b * POOL_ROWS : ((uint32_t)max(begins, 0) << d.page_shift) + (b & in_page) * POOL_ROWS;
        const uint32_t valid = begins < 0 || pos >= ask.len ? 0 : min(POOL_ROWS, ask.len - pos), stage = asked % SP_STAGES;
        held = (held & ~(255u << (8 * stage))) | valid << (8 * stage);
        if (valid != 0 && lane == 0) {
            mbar_expect_tx(bar + 8 * stage, B::BYTES);
            bulk_g2s(ring + stage * B::BYTES, p.a.pool.rows + ((((size_t)pg * d.kv_heads + ask.h) << bs) + (b & in_page)) * B::BYTES, B::BYTES, bar + 8 * stage);
        }
        ask.next += SP_WARPS;
        asked += 1;
    };
#pragma unroll 1
    for (uint32_t i = 0; i < SP_STAGES; ++i) request();
    float *s_factor = reinterpret_cast<float *>(smb + S::FACTOR), *s_join = reinterpret_cast<float *>(smb + S::JOIN);
    float2 *s_ml = reinterpret_cast<float2 *>(smb + S::ML);
    const LanePlaces<HD, BITS> place(lane);
    const Expand ex;
    Query<HD, QT, NR> q;
    State<HD, NR> st;
    bool ok = true;
    uint32_t i = 0;
    // items of the part
#pragma unroll 1
    for (;;) {
        put_queries<HD, QT, NR>(p, it, tid, smb + S::QUERY, s_factor);
        __syncthreads();
        get_queries<HD, QT, NR>(sbase + S::QUERY, sbase + S::FACTOR, lane, q);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) st.o[r][j][0] = st.o[r][j][1] = st.o[r][j][2] = st.o[r][j][3] = 0.0f;
            st.m[r][0] = st.m[r][1] = -INFINITY;
            st.l[r][0] = st.l[r][1] = 0.0f;
        }
        const uint32_t here = min(left, it.blocks - it.next);
        const bool whole = here == it.blocks;
        left -= here;
#pragma unroll 1
        for (uint32_t b = warp; b < here; b += SP_WARPS, ++i) {
            const uint32_t stage = i % SP_STAGES, valid = held >> (8 * stage) & 255u;
            if (valid != 0) {
                bool landed = mbar_try_wait(bar + 8 * stage, phase >> stage & 1u) != 0;
                for (uint32_t spin = 0; spin < WAIT_LIMIT && !landed; ++spin) landed = mbar_try_wait(bar + 8 * stage, phase >> stage & 1u) != 0;
                landed = __all_sync(0xffffffffu, landed);
                ok = ok && landed;
                phase ^= 1u << stage;
                block_step<HD, BITS, QT, PT, NR>(ring + stage * B::BYTES, valid, lane, place, ex, q, st);
            }
            __syncwarp();                          // all lanes are done with the stage
            request();
        }
        // the four warps' results, eight rows at a time; then HD / 8 threads have a row
        const uint32_t n = lane >> 2, t4 = lane & 3u, row = tid / (HD / 8), l = tid % (HD / 8);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            if (r > 0) __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) st.l[r][e] += __shfl_xor_sync(0xffffffffu, st.l[r][e], o);
                float *to = s_join + (warp * 8 + 2 * t4 + e) * S::PITCH + n * (HD / 8 / B::G);
#pragma unroll
                for (int j = 0; j < HD / 16; j += 2) *reinterpret_cast<float4 *>(to + (B::G == 2 && j >= 4 ? 64 + 2 * (j - 4) : 2 * j)) = make_float4(st.o[r][j][e], st.o[r][j][2 + e], st.o[r][j + 1][e], st.o[r][j + 1][2 + e]);
                if (n == 0) s_ml[warp * 8 + 2 * t4 + e] = make_float2(st.m[r][e], st.l[r][e]);
            }
            __syncthreads();
            if (row < 8) {                     // whole warps
                float m = -INFINITY, sum = 0.0f, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < (int)SP_WARPS; ++w) m = fmaxf(m, s_ml[w * 8 + row].x);
                const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
                for (int w = 0; w < (int)SP_WARPS; ++w) {
                    const float2 ml = s_ml[w * 8 + row];
                    const float f = exp2_approx(ml.x - base);
                    const float4 *from = reinterpret_cast<const float4 *>(s_join + (w * 8 + row) * S::PITCH + l * 8);
                    const float4 a = from[0], c = from[1];
                    sum = __fmaf_rn(f, ml.y, sum);
                    v[0] = __fmaf_rn(f, a.x, v[0]); v[1] = __fmaf_rn(f, a.y, v[1]); v[2] = __fmaf_rn(f, a.z, v[2]); v[3] = __fmaf_rn(f, a.w, v[3]);
                    v[4] = __fmaf_rn(f, c.x, v[4]); v[5] = __fmaf_rn(f, c.y, v[5]); v[6] = __fmaf_rn(f, c.z, v[6]); v[7] = __fmaf_rn(f, c.w, v[7]);
                }
                if (whole && p.a.prefix_len == 0) {
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] *= inv;
                    transform8_back(v, p.a.pool.signs[l / 4] >> (l % 4 * 8), lane);
                    uint32_t t, head;
                    if (item_row(p, it, 8 * r + row, t, head)) rows_put8(p.a.out, t * p.a.out.token_stride + head * p.a.out.head_stride + l * 8, v);
                } else if (8 * r + row < p.slot_rows(it.prefix)) {
                    const uint32_t rows = p.slot_rows(it.prefix);
                    float *slot = p.slot(it.prefix, unit, it.index), *o = slot + (8 * r + row) * HD + l * 8;
                    reinterpret_cast<float4 *>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
                    reinterpret_cast<float4 *>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
                    if (l == 0) *reinterpret_cast<float2 *>(slot + rows * HD + 2 * (8 * r + row)) = make_float2(m, sum);
                }
            }
        }
        if (left == 0) break;
        item_after(p, it);
    }
    if (!ok && lane == 0) atomicCAS(p.a.pool.err, 0u, 1u);
    if (behind) {
        pdl_wait();
        pdl_trigger();
    }
}

// ------------------------------------------------------------------------------------------------ partial results
// `ways` warps (1 .. 8) share a row (token, head): out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s, transformed back.  Items that one CTA
// finished are left alone.
constexpr uint32_t MERGE_WARPS = 8;
template <int HD> __global__ void __launch_bounds__(MERGE_WARPS * 32) pool_merge_kernel(const __grid_constant__ SplitArgs p, uint32_t ways) {
    constexpr int E = HD / 32;
    __shared__ float s_o[MERGE_WARPS][HD], s_l[MERGE_WARPS];
    __shared__ uint64_t s_sum[MERGE_WARPS][2];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kh = p.a.pool.d.kv_heads, group = p.a.heads / kh, rows_here = MERGE_WARPS / ways;
    const uint32_t all_rows = p.a.n_tok * p.a.heads, row0 = blockIdx.x * rows_here, id = min(all_rows - 1, row0 + warp / ways);
    const uint32_t t0 = row0 / p.a.heads, t = id / p.a.heads, head = id % p.a.heads, h = head / group, in = head % group;
    pdl_wait();
    pdl_trigger();
    // pieces of the prefix item, then of the token's own: [first, first + n) of the CTAs for each
    uint32_t near_first = 0, near_n = 0, near_item = 0, own_first = 0, own_n = 0;
    const uint32_t own_item = (t * kh + h) * p.rbo + in / p.tile, r = t * group + in;
    const uint64_t mine = item_blocks(p, t);
    if (p.pieces != 0) {
        const uint32_t part = piece_blocks(p.pieces, (uint32_t)mine);
        own_first = own_item * p.pieces;
        own_n = mine > 0 ? (uint32_t)((mine + part - 1) / part) : 0;
    } else {                                   // the CTA sums up to its first token, a warp the few up to its own
        uint64_t sum[2] = {0, 0};
        for (uint32_t k = threadIdx.x; k < p.a.n_tok; k += MERGE_WARPS * 32) {
            const uint32_t n = item_blocks(p, k);
            sum[0] += n;
            sum[1] += k < t0 ? n : 0;
        }
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) {
            sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], m);
            sum[1] += __shfl_xor_sync(0xffffffffu, sum[1], m);
        }
        if (lane == 0) { s_sum[warp][0] = sum[0]; s_sum[warp][1] = sum[1]; }
        __syncthreads();
        uint64_t total = 0, before = 0;
        for (uint32_t k = 0; k < MERGE_WARPS; ++k) { total += s_sum[k][0]; before += s_sum[k][1]; }
        for (uint32_t k = t0; k < t; ++k) before += item_blocks(p, k);
        if (mine > 0) {
            const uint64_t per = part_blocks(total * kh * p.rbo, p.units), b = before * kh * p.rbo + (uint64_t)(h * p.rbo + in / p.tile) * mine, e = b + mine;
            own_first = (uint32_t)(b / per);
            own_n = (uint32_t)((e - 1) / per) + 1 - own_first;
        }
    }
    if (p.near_units > 0) {
        near_item = h * p.rbp + r / p.tile;
        const uint32_t part = piece_blocks(p.near_pieces, prefix_blocks(p));
        near_first = near_item * p.near_pieces;
        near_n = (prefix_blocks(p) + part - 1) / part;
    }
    if (p.flash.on) {
        const FlashArgs &f = p.flash;
        near_item = h * f.row_tiles + r / (f.halved ? FLASH_ROWS : 2 * FLASH_ROWS);
        const uint32_t b = near_item * f.tiles, e = b + f.tiles;
        near_first = b / f.part;
        near_n = ((e - 1) / f.part + 1 - near_first) << (f.halved ? 1 : 0);
    }
    // an item without a block has one piece all the same, which has written its zeros
    const bool finished = p.a.prefix_len == 0 && (own_n == 1 || (p.pieces != 0 && own_n == 0));
    const uint32_t n = finished ? 0 : near_n + own_n;
    auto slot = [&](uint32_t i, uint32_t &row, uint32_t &rows) -> const float * {
        const bool near = i < near_n;
        if (near && p.flash.on) {             // two tiles of rows, or two streams over the same rows
            const uint32_t second = p.flash.halved ? i & 1u : r / FLASH_ROWS & 1u;
            row = r % FLASH_ROWS;
            rows = FLASH_ROWS;
            return p.near + (size_t)(near_first + (p.flash.halved ? i >> 1 : i) + near_item) * flash_slot_floats(HD) + second * (flash_slot_floats(HD) / 2);
        }
        row = (near ? r : in) % p.tile;
        rows = p.slot_rows(near);
        return near ? p.slot(true, near_first + i, near_item) : p.slot(false, own_first + i - near_n, own_item);
    };
    float top = -INFINITY;
    for (uint32_t i = lane; i < n; i += 32) {
        uint32_t row, rows;
        const float *s = slot(i, row, rows);
        top = fmaxf(top, __ldcg(s + rows * HD + 2 * row));
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    if (top == -INFINITY) top = 0.0f;
    float o[E], l = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = 0.0f;
#pragma unroll 4
    for (uint32_t i = warp % ways; i < n; i += ways) {
        uint32_t row, rows;
        const float *s = slot(i, row, rows);
        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(s + rows * HD) + row);
        float v[E];
        if constexpr (E == 4) {
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(s + row * HD) + lane);
            v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        } else {
            const float2 x = __ldcg(reinterpret_cast<const float2 *>(s + row * HD) + lane);
            v[0] = x.x; v[1] = x.y;
        }
        const float w = exp2_approx(ml.x - top);
        l = __fmaf_rn(w, ml.y, l);
#pragma unroll
        for (int k = 0; k < E; ++k) o[k] = __fmaf_rn(w, v[k], o[k]);
    }
#pragma unroll
    for (int k = 0; k < E; ++k) s_o[warp][lane * E + k] = o[k];
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    if (warp % ways != 0 || finished || row0 + warp / ways >= all_rows) return;
    l = 0.0f;
    const uint32_t c = lane % (HD / 8);        // eight elements a lane, every HD / 8 lanes alike
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (uint32_t w = warp; w < warp + ways; ++w) {
        l += s_l[w];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += s_o[w][c * 8 + i];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inv;
    transform8_back(v, p.a.pool.signs[c / 4] >> (c % 4 * 8), lane);
    if (lane < HD / 8) rows_put8(p.a.out, t * p.a.out.token_stride + head * p.a.out.head_stride + c * 8, v);
}

// ------------------------------------------------------------------------------------------------ launches
// A line of blocks in equal parts, or items in equal pieces, one a CTA?  A piece begins no second item, and nothing has to be looked up for it, but
// pieces are as equal as the items are long.  The prefix and chosen pages: items of one length, pieces.  Tables, by the widest row that the table
// has room for, in us of the whole call over ragged lengths (8 bits x 128 bf16; 4 x 64 fp16 and 4 x 128 fp32 draw the same lines):
//   * up to WHOLE blocks, unless a prefix has to be joined anyway, and from 16 items a resident CTA on, an item is one piece: 16 blocks x 48 / 192
//     items 6.4 / 7.9, cut in two 10.0 / 14.0 (a merge follows), as a line 18.5 / 26.5; 32 blocks x 96 / 192 items 9.3 / 10.5, in pieces 13.9 / 15.8 (32
//     blocks x 32 items behind a prefix, 4 bits: whole 93, in pieces 83);
//   * pieces of as many blocks as give CTAs that the SMs hold at once (a shorter item has fewer: the others leave at once), of LONGEST at most:
//     256 blocks x 48 items 21 in eight pieces, 47 whole, 26 as a line; 192 items 48 in two, 36 as a line;
//   * more items than that: whole up to 2 LONGEST blocks (2400 items of 4 / 64 / 128 blocks 23 / 70 / 117, as a line 65 / 110 / 161), a line from there
//     (1200 items of 512 blocks 221, whole 250; at 256 the two are alike).
constexpr uint32_t WHOLE = 32, LONGEST = 64;
uint32_t own_pieces(uint64_t items, uint64_t widest, uint64_t room, bool joined) {
    if ((widest <= WHOLE && !joined) || items >= 16 * room) return 1;
    for (uint64_t part = MIN_PART; part <= LONGEST; part *= 2)
        if (items * ((widest + part - 1) / part) <= room) return (uint32_t)((widest + part - 1) / part);
    return widest <= 2 * LONGEST ? 1 : 0;
}
SplitArgs split_plan(const PoolAttnArgs &a, uint32_t type) {
    SplitArgs p{};
    p.a = a;
    const PoolShape &d = a.pool.d;
    const uint32_t group = a.heads / d.kv_heads;
    const uint32_t rows = a.n_tok * group;
    // More rows than a tile of this kernel: k2t_pool_flash.cu, which expands a cached row once for 128 or 256 query rows where this one does for
    // 16.  Its start costs more, so it takes FLASH_WORK tiles of 16 rows x 16 positions and up.  Time here over time there for 24 to 384 rows of 1 to 8 kv
    // heads, widths 64 and 128, 8 and 4 bits, all types (the whole call; median, and the range that the shapes leave): below 1024 tiles 0.75
    // (0.63 .. 1.10), to 2048 0.84 (0.74 .. 0.97), to 8192 1.0 (0.87 .. 1.29), to 16384 1.0 (0.88 .. 1.35), above 1.39 (1.13 .. 2.67); the low ends are 24 or 32
    // rows, which fill a fifth of a tile, and fp32, the high ends 320 rows.
    constexpr uint64_t FLASH_WORK = 2048;
    p.flash.on = a.prefix_len > 0 && rows > 16 && (uint64_t)((rows + 15) / 16) * d.kv_heads * prefix_blocks(p) >= FLASH_WORK;
    if (p.flash.on) {
        FlashArgs &f = p.flash;
        f.halved = rows <= FLASH_ROWS || type != TYPE_BF16;
        f.row_tiles = f.halved ? (rows + FLASH_ROWS - 1) / FLASH_ROWS : (rows + 2 * FLASH_ROWS - 1) / (2 * FLASH_ROWS);
        f.items = d.kv_heads * f.row_tiles;
        f.tiles = (a.prefix_len + 63) / 64;
        f.part = (uint32_t)std::max<uint64_t>(FLASH_MIN_PART, ((uint64_t)f.items * f.tiles + a.sm_count - 1) / a.sm_count);
    }
    const bool near = a.prefix_len > 0 && !p.flash.on;
    p.tile = group > 8 || (near && rows > 8) ? 16 : 8;
    p.rbo = (group + p.tile - 1) / p.tile;
    p.rbp = near ? (rows + p.tile - 1) / p.tile : 0;
    const uint64_t items = (uint64_t)a.n_tok * d.kv_heads * p.rbo, room = (uint64_t)a.sm_count * split_ctas(d.head_dim, d.bits, type != TYPE_BF16, type == TYPE_F32, p.tile / 8);
    const auto pieces_of = [&](uint64_t n, uint64_t blocks) { return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(room / n, blocks / MIN_PART)); };
    if (near) {
        p.near_pieces = pieces_of((uint64_t)d.kv_heads * p.rbp, prefix_blocks(p));
        p.near_units = d.kv_heads * p.rbp * p.near_pieces;
    }
    p.pieces = a.chosen != nullptr ? pieces_of(items, (uint64_t)a.top << (d.page_shift - 4)) : own_pieces(items, std::max<uint64_t>(1, (uint64_t)a.pages_stride << (d.page_shift - 4)), room, a.prefix_len > 0);
    p.units = (uint32_t)(p.pieces != 0 ? items * p.pieces : room);
    return p;
}
size_t own_slots(const SplitArgs &p) { return p.units + (p.pieces != 0 ? 0 : (size_t)p.a.n_tok * p.a.pool.d.kv_heads * p.rbo); }
size_t near_floats(const SplitArgs &p) {
    if (p.flash.on) return ((size_t)p.a.sm_count + p.flash.items) * flash_slot_floats(p.a.pool.d.head_dim) + p.flash.items * flash_query_bytes(p.a.pool.d.head_dim) / 4;
    return p.near_units * (size_t)p.slot_floats(true);
}

// Halves of an operand: bf16 queries and weights are rounded to one each (11 bits where bf16 has 8); fp16 queries keep two, since a score is a
// sum of head_dim roundings (one: an output of fp16 rows 2.3 times as far from 64 bits as its own rounding); fp32 keeps two of both.
template <int HD, int BITS, int QT, int PT, int NR> cudaError_t split_go(cudaStream_t s, const SplitArgs &p) {
    constexpr size_t smem = SplitSmem<HD, BITS, QT, NR>::BYTES;
    static_assert((smem + 1024) * split_ctas(HD, BITS, QT == 2, PT == 2, NR) <= 233472, "shared memory of an SM");
    const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void *>(pool_split_kernel<HD, BITS, QT, PT, NR>), smem);
    if (e != cudaSuccess) return e;
    return launch_kernel(pool_split_kernel<HD, BITS, QT, PT, NR>, dim3(p.near_units + p.units), dim3(SP_WARPS * 32), smem, s, true, p);
}
template <int HD, int BITS, int NR> cudaError_t split_type(cudaStream_t s, const SplitArgs &p) {
    const uint32_t type = p.a.q.type;
    return type == TYPE_F32 ? split_go<HD, BITS, 2, 2, NR>(s, p) : type == TYPE_F16 ? split_go<HD, BITS, 2, 1, NR>(s, p) : split_go<HD, BITS, 1, 1, NR>(s, p);
}
template <int HD, int BITS> cudaError_t split_launch(cudaStream_t s, const SplitArgs &p) { return p.tile == 8 ? split_type<HD, BITS, 1>(s, p) : split_type<HD, BITS, 2>(s, p); }

}  // namespace

// Room for a call of these sizes whatever its table's width and choice (a line has the most partial results), and for one without a prefix.
size_t pool_work_bytes(const PoolShape &d, uint32_t heads, uint32_t n_tok, uint32_t prefix_len, uint32_t sm_count) {
    size_t most = 0;
    if (n_tok == 0) return 0;
    for (uint32_t type : {TYPE_F32, TYPE_BF16, TYPE_F16})
        for (uint32_t prefix : {0u, prefix_len}) {
            PoolAttnArgs a{};
            a.pool.d = d;
            a.heads = heads;
            a.n_tok = n_tok;
            a.prefix_len = prefix;
            a.sm_count = sm_count;
            a.pages_stride = 0x7fffffff;
            const SplitArgs p = split_plan(a, type);
            most = std::max(most, ((p.units + (size_t)n_tok * d.kv_heads * p.rbo) * p.slot_floats(false) + near_floats(p)) * 4);
        }
    return most;
}

cudaError_t launch_pool_attend(cudaStream_t s, const PoolAttnArgs &a, uint32_t *launched) {
    SplitArgs p = split_plan(a, a.q.type);
    p.own = reinterpret_cast<float *>(a.work);
    p.near = p.own + own_slots(p) * p.slot_floats(false);          // 16-byte boundaries: see slot_floats
    const PoolShape &d = a.pool.d;
    const bool b8 = d.bits == 8;
    cudaError_t e = cudaSuccess;
    if (p.flash.on) {
        p.flash.queries = reinterpret_cast<uint8_t *>(p.near + ((size_t)a.sm_count + p.flash.items) * flash_slot_floats(d.head_dim));
        p.flash.factors = reinterpret_cast<float *>(p.flash.queries + p.flash.items * (flash_query_bytes(d.head_dim) - 2 * FLASH_ROWS * 4));
        e = launch_pool_flash(s, p);
        if (e != cudaSuccess) return e;
        *launched += 2;
    }
    e = d.head_dim == 128 ? (b8 ? split_launch<128, 8>(s, p) : split_launch<128, 4>(s, p)) : b8 ? split_launch<64, 8>(s, p) : split_launch<64, 4>(s, p);
    *launched += 1;
    if (e != cudaSuccess || (p.pieces == 1 && a.prefix_len == 0)) return e;
    *launched += 1;
    // rows are few where their pieces are many
    const uint32_t rows = a.n_tok * a.heads;
    uint32_t ways = MERGE_WARPS;
    while (ways > 1 && (uint64_t)rows * ways > 4 * MERGE_WARPS * (uint64_t)a.sm_count) ways /= 2;
    const auto merge = d.head_dim == 128 ? pool_merge_kernel<128> : pool_merge_kernel<64>;
    return launch_kernel(merge, dim3((rows + MERGE_WARPS / ways - 1) / (MERGE_WARPS / ways)), dim3(MERGE_WARPS * 32), 0, s, true, p, ways);
}

}  // namespace k2t
