// Shared by the kernels of the pool's attention: how the work of a call is laid out in a line, and where partial results lie.
#pragma once
#include "k2t_kv_pool.h"

namespace k2t {

// The prefix over many rows (k2t_pool_flash.cu): items are (kv head, 2 FLASH_ROWS rows), tiles of 64 positions; a line of items * tiles, `part` of it
// a CTA.  halved: an item has FLASH_ROWS rows, and its tiles are dealt out to two streams over the same rows.
constexpr uint32_t FLASH_ROWS = 128, FLASH_MIN_PART = 2;          // tiles of a CTA at least (2 against 4: 24 against 25 us behind 2000 positions)
// Tiles of a call's line, and a part behind it, are counted in 32 bits; a part is at most a 64th of the line (SMs).
constexpr uint64_t MOST_TILES = (1ull << 32) - (1ull << 26);
struct FlashArgs {
    bool on, halved;
    uint32_t items, row_tiles, tiles, part;
    uint8_t *queries;            // operand tiles of all items, two of FLASH_ROWS rows each
    float *factors;              // of their rows
};
// bytes of an item's queries (at most two tiles: of rows, or of terms) and factors
__host__ __device__ constexpr size_t flash_query_bytes(uint32_t head_dim) { return 2 * FLASH_ROWS * (head_dim * 2 + 4); }
// partial results of a CTA and item: two of FLASH_ROWS rows
__host__ __device__ constexpr uint32_t flash_slot_floats(uint32_t head_dim) { return 2 * FLASH_ROWS * (head_dim + 2); }

// A partial result: rows x head_dim numerators, then (maximum, denominator) of each row.
struct SplitArgs {
    PoolAttnArgs a;
    uint32_t tile, rbo, rbp;     // query rows of a CTA, 8 or 16; tiles of a token and kv head; of the prefix (0: not in this kernel)
    uint32_t units, pieces;      // CTAs for own rows; of an item, or 0: the line of all items' blocks is cut into parts
    uint32_t near_units, near_pieces;          // CTAs for the prefix, before them; of an item
    float *own, *near;           // partial results of own rows; of the prefix
    FlashArgs flash;

    __host__ __device__ uint32_t slot_rows(bool prefix) const { const uint32_t g = a.heads / a.pool.d.kv_heads; return prefix || g > tile ? tile : g; }
    __host__ __device__ uint32_t slot_floats(bool prefix) const { return (slot_rows(prefix) * (a.pool.d.head_dim + 2) + 3u) & ~3u; }       // 16-byte boundaries
    // CTAs and items both ascend along the line, so their sum numbers the parts of items
    __host__ __device__ float *slot(bool prefix, uint32_t unit, uint32_t item) const {
        return (prefix ? near : own) + (size_t)(prefix || pieces != 0 ? unit : unit + item) * slot_floats(prefix);
    }
};
__host__ __device__ inline uint32_t prefix_blocks(const SplitArgs &p) { return (p.a.prefix_len + POOL_ROWS - 1) / POOL_ROWS; }
// blocks of a CTA's part: at least MIN_PART, since a part costs its queries and a partial result
constexpr uint32_t MIN_PART = 8;
__host__ __device__ inline uint64_t part_blocks(uint64_t all, uint32_t units) { const uint64_t n = (all + units - 1) / units; return n < MIN_PART ? MIN_PART : n; }

// blocks of a piece
__host__ __device__ inline uint32_t piece_blocks(uint32_t pieces, uint32_t blocks) { return blocks == 0 ? 1 : (blocks + pieces - 1) / pieces; }

cudaError_t launch_pool_flash(cudaStream_t s, const SplitArgs &p);

}  // namespace k2t
