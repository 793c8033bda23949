// Attention over the pool for few query rows at a time: tables of pages, chosen pages, and a shared prefix with up to a tile of rows.
//   score t_ij = (c_i q_i . code_j) ks_j, kept as x_ij = t_ij + log2 vs_j, so that 2^x is the weight already times the value's scale and
//   every operand of a product is a code (whole numbers up to 127, exact halves) or a weight of at most 2^8;
//   numerator O_i = sum_j 2^(x_ij - m_i) codev_j, denominator l_i = sum_j 2^(x_ij - m_i) / vs_j, with the running maximum m_i of x.
// Positions out of sight have ks = 0, log2 vs = -inf, 1 / vs = 0: no mask per element, and nothing of theirs is multiplied.
//
// A WARP is the unit of work.  It holds 16 query rows as operands in registers (m16n8k16, halves) and walks blocks of 16 positions, which
// a bulk copy each brings into a ring of its own; rows are queries of one kv head, so a cached row is read once for the heads that share
// it.  The blocks of all items (token, kv head) are one long line cut into equal parts, one per warp: ragged lengths and a single
// long sequence alike keep every warp busy to the end.  An item that lies in one part is finished there; the others leave partial
// results, which pool_merge_kernel joins.
#include <algorithm>

#include "k2t_flash_tc.cuh"
#include "k2t_kv_pool.cuh"
#include "k2t_pool_attn.h"

namespace k2t {
namespace {

constexpr uint32_t SP_WARPS = 4, SP_STAGES = 3, WAIT_LIMIT = 1u << 22;
// CTAs on an SM: registers (two for rows of 128 with queries in two halves)
template <int HD, int QT> struct SplitCtas { static constexpr uint32_t N = HD == 128 && QT == 2 ? 2 : 3; };
template <int HD, int BITS, int QT> constexpr uint32_t split_smem() { return SP_WARPS * (SP_STAGES * PoolBlock<HD, BITS>::BYTES + QT * HD / 16 * 512); }

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int WORDS> __device__ __forceinline__ void lds_words(uint32_t addr, uint32_t *w) {
    if constexpr (WORDS == 4) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
    else if constexpr (WORDS == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}

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

// One item of the line: its blocks are [begin, end) there.
struct Item {
    uint64_t begin, end;
    uint32_t index, t, h, rb;          // of the prefix items: (h, rb)
    uint32_t len;                      // positions in sight
    const int32_t *list;               // pages, or choices among the pages of `table`
    const int32_t *table;
    bool prefix;
};

__device__ __forceinline__ void item_fill(const SplitArgs &p, Item &it) {
    if (it.prefix) {
        it.list = p.a.prefix_pages;
        it.len = p.a.prefix_len;
        return;
    }
    int32_t seq;
    it.len = seen_rows(p.a, it.t, seq);
    it.table = p.a.pages + (size_t)max(seq, 0) * p.a.pages_stride;
    it.list = p.a.chosen != nullptr ? p.a.chosen + ((size_t)it.t * p.a.pool.d.kv_heads + it.h) * p.a.top : it.table;
}

// Sums of the tokens' blocks over a warp: the whole, and the place of the token that holds block `x` of them (counted per kv head and tile).
__device__ __forceinline__ uint64_t warp_total(const SplitArgs &p, uint32_t lane) {
    if (p.a.chosen != nullptr) return (uint64_t)p.a.n_tok * (p.a.top << (p.a.pool.d.page_shift - 4));
    uint64_t sum = 0;
    for (uint32_t t = lane; t < p.a.n_tok; t += 32) sum += item_blocks(p, t);
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    return sum;
}
__device__ __forceinline__ void warp_find(const SplitArgs &p, uint64_t x, uint32_t lane, uint32_t &t, uint64_t &before, uint32_t &blocks) {
    if (p.a.chosen != nullptr) {
        blocks = p.a.top << (p.a.pool.d.page_shift - 4);
        t = (uint32_t)(x / blocks);
        before = (uint64_t)t * blocks;
        return;
    }
    uint64_t base = 0;
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
    t = p.a.n_tok; before = base; blocks = 0;            // not reached: x lies below the total
}

// The item that holds block x of the line: prefix items first, then tokens in order, of a token its kv heads, of those their tiles.
__device__ __forceinline__ void item_at(const SplitArgs &p, uint64_t x, uint32_t lane, Item &it) {
    const uint64_t far = prefix_line(p);
    if (x < far) {
        const uint32_t nb = prefix_blocks(p);
        it.prefix = true;
        it.index = (uint32_t)(x / nb);
        it.h = it.index / p.rbp;
        it.rb = it.index % p.rbp;
        it.t = 0;
        it.begin = (uint64_t)it.index * nb;
        it.end = it.begin + nb;
    } else {
        const uint32_t per = p.a.pool.d.kv_heads * p.rbo;
        uint32_t blocks;
        uint64_t before;
        warp_find(p, (x - far) / per, lane, it.t, before, blocks);
        const uint32_t sub = (uint32_t)((x - far - before * per) / blocks);
        it.prefix = false;
        it.h = sub / p.rbo;
        it.rb = sub % p.rbo;
        it.index = it.t * per + sub;
        it.begin = far + before * per + (uint64_t)sub * blocks;
        it.end = it.begin + blocks;
    }
    item_fill(p, it);
}

// ------------------------------------------------------------------------------------------------ the warp's rows
// Query row i of an item: whether it exists, its token and head.
__device__ __forceinline__ bool item_row(const SplitArgs &p, const Item &it, uint32_t i, uint32_t &t, uint32_t &head) {
    const uint32_t group = p.a.heads / p.a.pool.d.kv_heads, r = it.rb * 16 + i;
    t = it.prefix ? r / group : it.t;
    head = it.h * group + (it.prefix ? r % group : r);
    return it.prefix ? t < p.a.n_tok : r < group;
}

// Sixteen consecutive elements from / to rows.
__device__ __forceinline__ void get16(const RowsArg &a, size_t at, float (&v)[16]) {
    rows_get8(a, at, *reinterpret_cast<float(*)[8]>(v));
    rows_get8(a, at + 8, *reinterpret_cast<float(*)[8]>(v + 8));
}

// Rows 'lane / 4' and that + 8: their elements [16 c, 16 c + 16) for c = t, and t + 4 where rows are 128 long; transformed, times a power
// of two that brings the largest to 2^13 .. 2^14 (so that both terms of a row are ordinary halves), as operand fragments: word 2 k + r
// of fragment i (and of its second term, HD / 16 further) for every lane, 16 bytes a lane.  They lie in shared memory: as 32 or 64
// registers they left room for two CTAs on an SM where there are three now.  c: factor of the scores of the two rows, in powers of two.
template <int HD, int QT> __device__ __forceinline__ void load_query(const SplitArgs &p, const Item &it, uint32_t lane, uint32_t *frags, float (&c)[2]) {
    const uint32_t n = lane >> 2, t4 = lane & 3u;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        uint32_t t, head;
        const bool live = item_row(p, it, n + 8 * r, t, head);
        float v[HD / 64][16], top = 0.0f;
#pragma unroll
        for (int g = 0; g < HD / 64; ++g) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[g][i] = 0.0f;
            if (live) get16(p.a.q, t * p.a.q.token_stride + head * p.a.q.head_stride + g * 64 + t4 * 16, v[g]);
            const uint32_t signs = p.a.pool.signs[2 * g + (t4 >> 1)] >> ((t4 & 1u) * 16);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[g][i] = __fmul_rn(flip(v[g][i], signs >> i & 1u), 0.125f);
            butterflies_in(v[g]);
            butterflies_across(v[g], 1, lane);
            butterflies_across(v[g], 2, lane);
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(v[g][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = query_exponent(top);
        const float up = power_of_two(e);
        c[r] = p.a.scale * LOG2E * power_of_two(-e);
#pragma unroll
        for (int g = 0; g < HD / 64; ++g)
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float x = v[g][4 * w + 2 * k] * up, y = v[g][4 * w + 2 * k + 1] * up;
                    const uint32_t hi = half2_bits(x, y);
                    frags[((4 * g + w) * 32 + lane) * 4 + r + 2 * k] = hi;
                    if constexpr (QT == 2) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                        frags[((HD / 16 + 4 * g + w) * 32 + lane) * 4 + r + 2 * k] = half2_bits(x - f.x, y - f.y);
                    }
                }
    }
}

template <int HD> struct State {
    float o[HD / 8][4], m[2], l[2];
};

// One block of 16 positions, `valid` of them in sight, at shared address `at`.
template <int HD, int BITS, int QT, int PT>
__device__ __forceinline__ void block_step(uint32_t at, uint32_t valid, uint32_t lane, uint32_t frags, const float (&c)[2], State<HD> &st) {
    using B = PoolBlock<HD, BITS>;
    constexpr int G = B::G;
    const uint32_t n = lane >> 2, t = lane & 3u;
    // scores of positions 4 (n / 2) + n % 2 (first tile of columns) and two further (second), per group of 64 elements
    float s[G][2][4];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int j = 0; j < 2; ++j) s[g][j][0] = s[g][j][1] = s[g][j][2] = s[g][j][3] = 0.0f;
#pragma unroll
    for (int g = 0; g < HD / 64; ++g) {
        uint32_t w[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t row = 4 * (n >> 1) + (n & 1u) + 2 * j;
            if (BITS == 8) {
                lds_words<4>(at + row_place<B::RB>(row, g * 64 + t * 16), w[j]);
            } else {
                uint32_t x[2];
                lds_words<2>(at + row_place<B::RB>(row, g * 32 + t * 8), x);
#pragma unroll
                for (int i = 0; i < 2; ++i) { w[j][2 * i] = centroids4(x[i]); w[j][2 * i + 1] = centroids4(x[i] >> 16); }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t a[QT][4];
#pragma unroll
            for (int k = 0; k < QT; ++k) lds_words<4>(frags + ((k * (HD / 16) + 4 * g + i) * 32 + lane) * 16, a[k]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t b0 = halves_lo(w[j][i]), b1 = halves_hi(w[j][i]);
#pragma unroll
                for (int k = 0; k < QT; ++k) mma_f16(s[G == 1 ? 0 : g][j], a[k], b0, b1);
            }
        }
    }
    // the lane's columns are positions 4 t .. 4 t + 3
    float ks[G][4], lv[4], iv[4], part[G][4];
    if (BITS == 8) {
        const float4 a = lds_f32x4(at + B::KS_AT + t * 16), b = lds_f32x4(at + B::VS_AT + t * 16);
        const float va[4] = {b.x, b.y, b.z, b.w};
        ks[0][0] = a.x; ks[0][1] = a.y; ks[0][2] = a.z; ks[0][3] = a.w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = va[i] == 0.0f ? 1.0f : va[i];          // a row of zeros: its codes are 0 as well
            lv[i] = __log2f(v);
            iv[i] = __fdividef(1.0f, v);
        }
    } else {
        uint32_t a[2 * G], b[2 * G];
        lds_words<2 * G>(at + B::KS_AT + t * 8 * G, a);
        lds_words<2 * G>(at + B::VS_AT + t * 8 * G, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v[G], top = 0.0f;                // scales are not negative, and all groups of a row are NaN or none
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int e = i * G + g;
                ks[g][i] = __uint_as_float(e & 1 ? a[e / 2] & 0xFFFF0000u : a[e / 2] << 16);
                v[g] = __uint_as_float(e & 1 ? b[e / 2] & 0xFFFF0000u : b[e / 2] << 16);
                top = fmaxf(top, v[g]);
            }
            const float u = v[0] != v[0] ? v[0] : top == 0.0f ? 1.0f : top;
            lv[i] = __log2f(u);
            iv[i] = __fdividef(1.0f, u);
#pragma unroll
            for (int g = 0; g < G; ++g) part[g][i] = v[g] * iv[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (4 * t + i >= valid) {
#pragma unroll
            for (int g = 0; g < G; ++g) { ks[g][i] = 0.0f; part[g][i] = 0.0f; }
            lv[i] = -INFINITY;
            iv[i] = 0.0f;
        }
    float x[2][4];                     // row, position
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float d = s[0][i >> 1][2 * r + (i & 1)] * ks[0][i];
            if (G == 2) d = __fmaf_rn(s[G - 1][i >> 1][2 * r + (i & 1)], ks[G - 1][i], d);
            x[r][i] = __fmaf_rn(d, c[r], lv[i]);
        }
    const float top0 = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), top1 = fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3]));
    // the maximum follows only where it has grown by more than 2^8: weights stay within halves, sums are exact in either case
    if (__any_sync(0xffffffffu, top0 > st.m[0] + 8.0f || top1 > st.m[1] + 8.0f)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float top = r == 0 ? top0 : top1;
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float m = fmaxf(st.m[r], top), al = m == -INFINITY ? 1.0f : exp2_approx(st.m[r] - m);
            st.m[r] = m;
            st.l[r] *= al;
#pragma unroll
            for (int j = 0; j < HD / 8; ++j) { st.o[j][2 * r] *= al; st.o[j][2 * r + 1] *= al; }
        }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const float m = st.m[r] == -INFINITY ? 0.0f : st.m[r];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[r][i] = exp2_approx(x[r][i] - m);
            st.l[r] = __fmaf_rn(x[r][i], iv[i], st.l[r]);
        }
    }
    uint32_t a[G][PT][4];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int k = 0; k < 4; ++k) {          // fragment word k: row k & 1, positions 2 (k / 2) and the next
            float u = x[k & 1][k & 2], v = x[k & 1][(k & 2) + 1];
            if (BITS == 4) { u *= part[g][k & 2]; v *= part[g][(k & 2) + 1]; }
            a[g][0][k] = half2_bits(u, v);
            if constexpr (PT == 2) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&a[g][0][k]));
                a[g][1][k] = half2_bits(u - f.x, v - f.y);
            }
        }
    // values of positions 4 t .. 4 t + 3; column n of tile j is element n HD / 8 + j
    constexpr int W = HD / 32;                 // words of four elements
    uint32_t v[4][W];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t from = at + B::V_AT + row_place<B::RB>(4 * t + i, n * (B::RB / 8));
        if (BITS == 8) {
            lds_words<W>(from, v[i]);
        } else {
            uint32_t y[W / 2];
            lds_words<W / 2>(from, y);
#pragma unroll
            for (int k = 0; k < W / 2; ++k) { v[i][2 * k] = centroids4(y[k]); v[i][2 * k + 1] = centroids4(y[k] >> 16); }
        }
    }
    // element j lies in group 0 where n HD / 8 < 64: lanes of one tile hold columns of both groups, so a tile is multiplied for each
    // group's weights into its own half of the columns -- by lanes' values set to zero outside the group
#pragma unroll
    for (int k = 0; k < W; ++k) {
        const uint32_t lo01 = prmt(v[0][k], v[1][k], 0x5140u), lo23 = prmt(v[2][k], v[3][k], 0x5140u), hi01 = prmt(v[0][k], v[1][k], 0x7362u), hi23 = prmt(v[2][k], v[3][k], 0x7362u);
        const uint32_t b0[4] = {halves_lo(lo01), halves_hi(lo01), halves_lo(hi01), halves_hi(hi01)};
        const uint32_t b1[4] = {halves_lo(lo23), halves_hi(lo23), halves_lo(hi23), halves_hi(hi23)};
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t x0 = G == 1 || (n >> 2) == (uint32_t)g ? b0[e] : 0u, x1 = G == 1 || (n >> 2) == (uint32_t)g ? b1[e] : 0u;
#pragma unroll
                for (int y = 0; y < PT; ++y) mma_f16(st.o[4 * k + e], a[g][y], x0, x1);
            }
    }
}

// The rows of a finished item, normalised and transformed back: the lane holds, of rows n and n + 8, elements (2 t + b) HD / 8 + j.
template <int HD> __device__ __forceinline__ void write_rows(const SplitArgs &p, const Item &it, uint32_t lane, const State<HD> &st) {
    constexpr int E = HD / 8;                  // consecutive elements of a lane
    const uint32_t n = lane >> 2, t4 = lane & 3u;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        uint32_t t, head;
        const bool live = item_row(p, it, n + 8 * r, t, head);
        const float inv = st.l[r] == 0.0f ? 0.0f : 1.0f / st.l[r];
        float v[2 * E];
#pragma unroll
        for (int j = 0; j < E; ++j) { v[j] = st.o[j][2 * r] * inv; v[E + j] = st.o[j][2 * r + 1] * inv; }
        butterflies_in(v);
        butterflies_across(v, 1, lane);
        if (HD == 64) butterflies_across(v, 2, lane);
        const uint32_t at = 2 * t4 * E, signs = p.a.pool.signs[at >> 5] >> (at & 31u);
#pragma unroll
        for (int i = 0; i < 2 * E; ++i) v[i] = flip(v[i] * 0.125f, signs >> i & 1u);
        if (live)
#pragma unroll
            for (int i = 0; i < 2 * E; i += 8)
                rows_put8(p.a.out, t * p.a.out.token_stride + head * p.a.out.head_stride + at + i, *reinterpret_cast<const float(*)[8]>(v + i));
    }
}

// Copies of blocks into the warp's ring, ahead of the steps: the item and block to ask for next, and 32 pages of its list over the lanes.
struct Requests {
    Item it;
    uint64_t x, end;           // next block of the line, end of the warp's part
    int32_t page, first;       // the lane's page of the list and the position it begins at (of a chosen one; else unused)
    uint32_t asked;            // blocks asked for
};

template <int HD, int BITS, int QT, int PT>
__global__ void __launch_bounds__(SP_WARPS * 32, SplitCtas<HD, QT>::N) pool_split_kernel(const __grid_constant__ SplitArgs p) {
    using B = PoolBlock<HD, BITS>;
    extern __shared__ __align__(128) uint8_t smb[];
    __shared__ __align__(8) uint64_t bars[SP_WARPS][SP_STAGES];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, unit = blockIdx.x * SP_WARPS + warp;
    uint32_t *frags = reinterpret_cast<uint32_t *>(smb + warp * (QT * HD / 16 * 512));
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smb) + SP_WARPS * (QT * HD / 16 * 512) + warp * SP_STAGES * B::BYTES, bar = (uint32_t)__cvta_generic_to_shared(bars[warp]);
    const PoolShape &d = p.a.pool.d;
    const uint32_t bs = d.page_shift - 4;
    if (lane == 0) {
        for (uint32_t i = 0; i < SP_STAGES; ++i) mbar_init(bar + 8 * i, 1);
        fence_mbar_init();
    }
    __syncwarp();
    pdl_wait();
    pdl_trigger();
    Requests rq;
    rq.asked = 0;
    if (p.direct) {             // the warp's part is one item, which may hold no block at all
        const uint32_t per = d.kv_heads * p.rbo;
        if (unit >= p.a.n_tok * per) return;
        rq.it.prefix = false;
        rq.it.index = unit;
        rq.it.t = unit / per;
        rq.it.h = unit % per / p.rbo;
        rq.it.rb = unit % p.rbo;
        rq.it.begin = rq.x = 0;
        item_fill(p, rq.it);
        rq.it.end = rq.end = p.a.chosen != nullptr ? p.a.top << bs : (rq.it.len + POOL_ROWS - 1) / POOL_ROWS;
    } else {
        const uint64_t all = prefix_line(p) + warp_total(p, lane) * d.kv_heads * p.rbo, per = part_blocks(all, p.units);
        rq.x = (uint64_t)unit * per;
        rq.end = min(all, rq.x + per);
        if (rq.x >= rq.end) return;
        item_at(p, rq.x, lane, rq.it);
    }
    Item it = rq.it;
    const uint64_t start = rq.x, end = rq.end;
    uint64_t x = start;
    uint32_t held = 0, phase = 0;              // a byte per stage: positions in sight; a bit per stage: parity of its next copy
    bool fresh = true;                         // the lanes' pages are to be read

    auto request = [&]() {                     // one block, into stage asked % SP_STAGES
        if (rq.x >= rq.end) return;
        if (rq.x >= rq.it.end) { item_at(p, rq.x, lane, rq.it); fresh = true; }
        const uint32_t b = (uint32_t)(rq.x - rq.it.begin), entry = b >> bs;
        if (fresh || (b & ((32u << bs) - 1u)) == 0) {
            fresh = false;
            const uint32_t e = (entry & ~31u) + lane, pages = (rq.it.len + (1u << d.page_shift) - 1) >> d.page_shift;
            rq.page = -1;
            rq.first = 0;
            if (rq.it.prefix || p.a.chosen == nullptr) {
                if (e < pages) rq.page = __ldcg(rq.it.list + e);
                else rq.page = 0;
            } else {
                const int32_t c = e < p.a.top ? __ldcg(rq.it.list + e) : -1;
                if (c >= 0 && (uint32_t)c < pages) { rq.page = __ldcg(rq.it.table + c); rq.first = c; }
                else { rq.page = 0; rq.first = -1; }
            }
            if (rq.page < 0 || (uint32_t)rq.page >= d.num_pages) { pool_bad_page(p.a.pool); rq.page = 0; rq.first = -1; }
        }
        const int32_t page = __shfl_sync(0xffffffffu, rq.page, entry & 31u), first = __shfl_sync(0xffffffffu, rq.first, entry & 31u);
        const bool listed = rq.it.prefix || p.a.chosen == nullptr;
        const uint64_t pos = listed ? (uint64_t)b * POOL_ROWS : ((uint64_t)max(first, 0) << d.page_shift) + (uint64_t)(b & ((1u << bs) - 1u)) * POOL_ROWS;
        const uint32_t valid = first < 0 || pos >= rq.it.len ? 0 : (uint32_t)min((uint64_t)POOL_ROWS, rq.it.len - pos), stage = rq.asked % SP_STAGES;
        held = (held & ~(255u << (8 * stage))) | valid << (8 * stage);
        if (valid != 0 && lane == 0) {
            mbar_expect_tx(bar + 8 * stage, B::BYTES);
            bulk_g2s(ring + stage * B::BYTES, p.a.pool.rows + (((size_t)page * d.kv_heads + rq.it.h << bs) + (b & ((1u << bs) - 1u))) * B::BYTES, B::BYTES, bar + 8 * stage);
        }
        rq.x += 1;
        rq.asked += 1;
    };
    for (uint32_t i = 0; i < SP_STAGES; ++i) request();
    float c[2];
    State<HD> st;
    auto begin = [&]() {
        load_query<HD, QT>(p, it, lane, frags, c);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) st.o[j][0] = st.o[j][1] = st.o[j][2] = st.o[j][3] = 0.0f;
        st.m[0] = st.m[1] = -INFINITY;
        st.l[0] = st.l[1] = 0.0f;
    };
    auto finish = [&]() {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 1);
            st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 2);
        }
        if (p.a.prefix_len == 0 && it.begin >= start && it.end <= end) { write_rows(p, it, lane, st); return; }
        float *slot = p.slot(it.prefix, unit, it.index);
        const uint32_t n = lane >> 2, t4 = lane & 3u, rows = p.slot_rows(it.prefix);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t row = n + 8 * r;
            if (row >= rows) continue;
            float *o = slot + row * HD + 2 * t4 * (HD / 8);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < HD / 8; j += 4)
                    *reinterpret_cast<float4 *>(o + b * (HD / 8) + j) = make_float4(st.o[j][2 * r + b], st.o[j + 1][2 * r + b], st.o[j + 2][2 * r + b], st.o[j + 3][2 * r + b]);
            if (t4 == 0) *reinterpret_cast<float2 *>(slot + rows * HD + 2 * row) = make_float2(st.m[r], st.l[r]);
        }
    };
    begin();
    bool ok = true;
    for (uint32_t i = 0; x < end; ++i, ++x) {
        if (x >= it.end) {
            finish();
            item_at(p, x, lane, it);
            begin();
        }
        const uint32_t stage = i % SP_STAGES, valid = held >> (8 * stage) & 255u;
        if (valid != 0) {
            bool landed = mbar_try_wait(bar + 8 * stage, phase >> stage & 1u) != 0;
            for (uint32_t spin = 0; spin < WAIT_LIMIT && !landed; ++spin) landed = mbar_try_wait(bar + 8 * stage, phase >> stage & 1u) != 0;
            landed = __all_sync(0xffffffffu, landed);
            ok = ok && landed;
            phase ^= 1u << stage;
            block_step<HD, BITS, QT, PT>(ring + stage * B::BYTES, valid, lane, (uint32_t)__cvta_generic_to_shared(frags), c, st);
        }
        __syncwarp();                          // all lanes are done with the stage
        request();
    }
    finish();
    if (!ok && lane == 0) atomicCAS(p.a.pool.err, 0u, 1u);
}

// ------------------------------------------------------------------------------------------------ partial results
// CTA = (token, head).  out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s, transformed back.  Items that one warp finished are left alone.
constexpr uint32_t MERGE_WARPS = 4;
template <int HD> __global__ void __launch_bounds__(MERGE_WARPS * 32) pool_merge_kernel(const __grid_constant__ SplitArgs p) {
    constexpr int E = HD / 32;
    __shared__ float s_o[MERGE_WARPS][HD], s_l[MERGE_WARPS];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kh = p.a.pool.d.kv_heads, group = p.a.heads / kh;
    const uint32_t t = blockIdx.x / p.a.heads, head = blockIdx.x % p.a.heads, h = head / group, in = head % group;
    pdl_wait();
    pdl_trigger();
    // pieces of the prefix item, then of the token's own: [first, last) of the warps for each
    uint32_t near_first = 0, near_n = 0, near_item = 0, own_first = 0, own_n = 0;
    const uint32_t own_item = (t * kh + h) * p.rbo + in / 16, r = t * group + in;
    if (p.direct) {
        own_n = item_blocks(p, t) > 0 ? 1 : 0;
    } else {
        uint64_t total = 0, before = 0;
        const uint64_t mine = item_blocks(p, t);
        if (p.a.chosen != nullptr) {
            total = p.a.n_tok * mine;
            before = t * mine;
        } else {
            for (uint32_t k = lane; k < p.a.n_tok; k += 32) {
                const uint32_t n = item_blocks(p, k);
                total += n;
                before += k < t ? n : 0;
            }
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) {
                total += __shfl_xor_sync(0xffffffffu, total, m);
                before += __shfl_xor_sync(0xffffffffu, before, m);
            }
        }
        const uint64_t far = prefix_line(p), per = part_blocks(far + total * kh * p.rbo, p.units);
        if (far > 0 && !p.flash.on) {
            near_item = h * p.rbp + r / 16;
            const uint64_t b = (uint64_t)near_item * prefix_blocks(p), e = b + prefix_blocks(p);
            near_first = (uint32_t)(b / per);
            near_n = (uint32_t)((e - 1) / per) + 1 - near_first;
        }
        if (mine > 0) {
            const uint64_t b = far + before * kh * p.rbo + (uint64_t)(h * p.rbo + in / 16) * mine, e = b + mine;
            own_first = (uint32_t)(b / per);
            own_n = (uint32_t)((e - 1) / per) + 1 - own_first;
            if (own_n == 1 && p.a.prefix_len == 0) return;
        }
    }
    if (p.flash.on) {
        const FlashArgs &f = p.flash;
        near_item = h * f.row_tiles + (f.halved ? 0u : r / (2 * FLASH_ROWS));
        const uint32_t b = near_item * f.tiles, e = b + f.tiles;
        near_first = b / f.part;
        near_n = ((e - 1) / f.part + 1 - near_first) << (f.halved ? 1 : 0);
    }
    const uint32_t n = near_n + own_n;
    auto slot = [&](uint32_t i, uint32_t &row, uint32_t &rows) -> const float * {
        const bool near = i < near_n;
        if (near && p.flash.on) {             // two tiles of rows, or two streams over the same rows
            const uint32_t second = p.flash.halved ? i & 1u : r / FLASH_ROWS & 1u;
            row = r % FLASH_ROWS;
            rows = FLASH_ROWS;
            return p.near + (size_t)(near_first + (p.flash.halved ? i >> 1 : i) + near_item) * flash_slot_floats(HD) + second * (flash_slot_floats(HD) / 2);
        }
        row = near ? r % 16 : in % 16;
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
    for (uint32_t i = warp; i < n; i += MERGE_WARPS) {
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
    if (warp != 0) return;
    float v[8];
    if (lane >= HD / 8) return;
    l = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = ((s_o[0][lane * 8 + i] + s_o[1][lane * 8 + i]) + (s_o[2][lane * 8 + i] + s_o[3][lane * 8 + i])) * inv;
    butterflies_in(v);
    constexpr uint32_t LANES = HD / 8, MASK = LANES == 16 ? 0xFFFFu : 0xFFu;
#pragma unroll
    for (uint32_t m = 1; m < 8; m <<= 1) {
        const bool upper = (lane & m) != 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = __shfl_xor_sync(MASK, v[i], m);
            v[i] = upper ? y - v[i] : v[i] + y;
        }
    }
    const uint32_t signs = p.a.pool.signs[lane / 4] >> (lane % 4 * 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = flip(v[i] * 0.125f, signs >> i & 1u);
    rows_put8(p.a.out, t * p.a.out.token_stride + head * p.a.out.head_stride + lane * 8, v);
}

// ------------------------------------------------------------------------------------------------ launches
// One warp per item where there are several items for every warp that the SMs hold: their ends then overlap anyway, and nothing has to
// be looked up or joined.
SplitArgs split_plan(const PoolAttnArgs &a, uint32_t type) {
    SplitArgs p{};
    p.a = a;
    const PoolShape &d = a.pool.d;
    const uint32_t group = a.heads / d.kv_heads;
    const uint64_t items = (uint64_t)a.n_tok * d.kv_heads * ((group + 15) / 16), room = (uint64_t)a.sm_count * (d.head_dim == 128 && type != TYPE_BF16 ? SplitCtas<128, 2>::N : SplitCtas<128, 1>::N) * SP_WARPS;
    p.rbo = (group + 15) / 16;
    const uint32_t rows = a.n_tok * group;
    p.flash.on = a.prefix_len > 0 && rows > 16;          // more than one tile of this kernel: k2t_pool_flash.cu
    if (p.flash.on) {
        FlashArgs &f = p.flash;
        f.halved = rows <= FLASH_ROWS;
        f.row_tiles = (rows + 2 * FLASH_ROWS - 1) / (2 * FLASH_ROWS);
        f.items = d.kv_heads * f.row_tiles;
        f.tiles = (a.prefix_len + 63) / 64;
        f.part = (uint32_t)std::max<uint64_t>(FLASH_MIN_PART, ((uint64_t)f.items * f.tiles + a.sm_count - 1) / a.sm_count);
    }
    p.rbp = a.prefix_len == 0 || p.flash.on ? 0 : (rows + 15) / 16;
    p.direct = p.rbp == 0 && items >= 4 * room;
    p.units = (uint32_t)(p.direct ? items : room);
    return p;
}
size_t own_slots(const SplitArgs &p) { return p.direct ? p.units : p.units + (size_t)p.a.n_tok * p.a.pool.d.kv_heads * p.rbo; }
size_t near_floats(const SplitArgs &p) {
    if (p.flash.on) return ((size_t)p.a.sm_count + p.flash.items) * flash_slot_floats(p.a.pool.d.head_dim);
    return p.rbp == 0 ? 0 : (p.units + (size_t)p.a.pool.d.kv_heads * p.rbp) * p.slot_floats(true);
}

// Halves of an operand: bf16 queries and weights are rounded to one each (11 bits where bf16 has 8); fp16 queries keep two, since a score is a
// sum of head_dim roundings (one: an output of fp16 rows 2.3 times as far from 64 bits as its own rounding); fp32 keeps two of both.
template <int HD, int BITS, int QT, int PT> cudaError_t split_go(cudaStream_t s, const SplitArgs &p) {
    const size_t smem = split_smem<HD, BITS, QT>();
    const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void *>(pool_split_kernel<HD, BITS, QT, PT>), smem);
    if (e != cudaSuccess) return e;
    return launch_kernel(pool_split_kernel<HD, BITS, QT, PT>, dim3((p.units + SP_WARPS - 1) / SP_WARPS), dim3(SP_WARPS * 32), smem, s, true, p);
}
template <int HD, int BITS> cudaError_t split_launch(cudaStream_t s, const SplitArgs &p) {
    const uint32_t type = p.a.q.type;
    return type == TYPE_F32 ? split_go<HD, BITS, 2, 2>(s, p) : type == TYPE_F16 ? split_go<HD, BITS, 2, 1>(s, p) : split_go<HD, BITS, 1, 1>(s, p);
}

}  // namespace

size_t pool_work_bytes(const PoolShape &d, uint32_t heads, uint32_t n_tok, uint32_t prefix_len, uint32_t sm_count) {
    PoolAttnArgs a{};
    a.pool.d = d;
    a.heads = heads;
    a.n_tok = n_tok;
    a.prefix_len = prefix_len;
    a.sm_count = sm_count;
    size_t most = 0;
    for (uint32_t type : {TYPE_F32, TYPE_BF16, TYPE_F16}) {
        const SplitArgs p = split_plan(a, type);
        most = std::max(most, (own_slots(p) * p.slot_floats(false) + near_floats(p)) * 4);
    }
    return most;
}

cudaError_t launch_pool_attend(cudaStream_t s, const PoolAttnArgs &a, uint32_t *launched) {
    SplitArgs p = split_plan(a, a.q.type);
    p.own = reinterpret_cast<float *>(a.work);
    p.near = p.own + own_slots(p) * p.slot_floats(false);
    const PoolShape &d = a.pool.d;
    const bool b8 = d.bits == 8;
    cudaError_t e = cudaSuccess;
    if (p.flash.on) {
        e = launch_pool_flash(s, p);
        if (e != cudaSuccess) return e;
        *launched += 1;
    }
    e = d.head_dim == 128 ? (b8 ? split_launch<128, 8>(s, p) : split_launch<128, 4>(s, p)) : b8 ? split_launch<64, 8>(s, p) : split_launch<64, 4>(s, p);
    *launched += 1;
    if (e != cudaSuccess || (p.direct && a.prefix_len == 0)) return e;
    *launched += 1;
    const auto merge = d.head_dim == 128 ? pool_merge_kernel<128> : pool_merge_kernel<64>;
    return launch_kernel(merge, dim3(a.n_tok * a.heads), dim3(MERGE_WARPS * 32), 0, s, true, p);
}

}  // namespace k2t
