// A pool of cached keys and values shared by many sequences (KronosCudaKvPool): geometry, arguments and launches of its operators.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>
#include <string>

#include "../../include/kronos_cuda_ffi.h"

namespace k2t {

constexpr uint32_t POOL_ROWS = 16;         // positions of a block, the unit of storage: their rows of keys, rows of values, scales

struct PoolShape {
    uint32_t kv_heads, head_dim, bits, page_shift, num_pages;          // page = 1 << page_shift positions
    bool block_keys;
    __host__ __device__ uint32_t row_bytes() const { return bits == 8 ? head_dim : head_dim / 2; }
    __host__ __device__ uint32_t scale_bytes() const { return bits == 8 ? 64 : head_dim / 2; }       // of a block's keys (or values)
    __host__ __device__ uint32_t block_bytes() const { return 2 * (POOL_ROWS * row_bytes() + scale_bytes()); }
    size_t rows_bytes() const { return ((size_t)num_pages << page_shift) / POOL_ROWS * kv_heads * block_bytes(); }
    size_t key_bytes() const { return block_keys ? (size_t)num_pages * kv_heads * head_dim : 0; }
    size_t key_scale_bytes() const { return block_keys ? (size_t)num_pages * kv_heads * 4 : 0; }
};

// What the kernels are handed of a pool.  signs: bit i = the sign of element i of a rotated row.
struct PoolView {
    PoolShape d;
    uint8_t *rows;               // [page][kv head][block of 16 positions]
    int8_t *block_keys;          // [page][kv head][head_dim]
    float *block_key_scales;     // [page][kv head]
    uint32_t signs[4];
    uint32_t *err;
};

// Rows [token][head][head_dim] of type f32 / bf16 / f16 (KRONOS_CUDA_TYPE_*); strides in elements.
struct RowsArg {
    void *p;
    uint64_t token_stride, head_stride;
    uint32_t type;
    bool wide;                   // eight elements of a row can be moved as 16-byte words
};

struct PoolStoreArgs {
    PoolView pool;
    RowsArg k, v;
    const int64_t *slots;
    uint32_t n_tok;              // times 2 kv heads: below 2^31
    uint32_t rows_mul, rows_shift, sm_count;
};
cudaError_t launch_pool_store(cudaStream_t s, const PoolStoreArgs &a, uint32_t *launched);
cudaError_t launch_pool_load(cudaStream_t s, const PoolStoreArgs &a, uint32_t *launched);

struct PoolAttnArgs {
    PoolView pool;
    RowsArg q, out;
    uint32_t n_tok, heads;
    const int32_t *lens, *seq, *pages;       // seq may be null: token t reads row t of the table
    uint32_t pages_stride;
    const int32_t *prefix_pages;
    uint32_t prefix_len;
    float scale;
    int32_t *chosen;                         // [token][kv head][top], or null
    uint32_t top, sinks, local;
    uint8_t *work;
    uint32_t sm_count;
};
cudaError_t launch_pool_attend(cudaStream_t s, const PoolAttnArgs &a, uint32_t *launched);
cudaError_t launch_pool_select(cudaStream_t s, const PoolAttnArgs &a, uint32_t *launched);
// of either attention over n_tok tokens, for sizes that are not refused; 0 for those that are
size_t pool_work_bytes(const PoolShape &d, uint32_t heads, uint32_t n_tok, uint32_t prefix_len, uint32_t sm_count);
size_t pool_workspace(const PoolShape &d, uint32_t heads, uint32_t n_tok, uint32_t prefix_len, uint32_t sm_count);

// Argument checks that need no device: false and a message.
enum { POOL_ATTEND = 0, POOL_CHOSEN = 1, POOL_SELECT = 2 };
bool pool_shape(const KronosCudaKvPoolConfig &c, PoolShape &d, std::string &why);
bool pool_rows(const PoolShape &d, uint32_t type, uint32_t heads, size_t n_tok, const KronosCudaRows &r, const char *name, bool written, RowsArg &out, std::string &why);
bool pool_attention(const PoolShape &d, const KronosCudaPoolAttention &c, int what, uint32_t sm_count, PoolAttnArgs &a, std::string &why);

}  // namespace k2t

struct KronosCudaKvPool {
    k2t::PoolView view;
    int device;
    uint32_t sm_count;
    size_t bytes;
};
