// C ABI of the shared pool of cached keys and values (include/kronos_cuda_ffi.h): handles, argument checks, calls.
#include <new>

#include "k2t_context.h"
#include "k2t_kv_pool.h"
#include "k2t_pool_attn.h"

namespace k2t {

// SplitMix64 sign of element i of 64-block `block` (rademacher_sign_masks_64, src/kernels/hadamard.rs:29-44)
static uint32_t sign_bit(uint64_t block, uint32_t i) {
    const uint64_t G = 0x9E3779B97F4A7C15ull;
    uint64_t z = G + block * 0xBF58476D1CE4E5B9ull + (uint64_t)(i + 1) * G;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return (uint32_t)((z ^ (z >> 31)) & 1ull);
}

bool pool_shape(const KronosCudaKvPoolConfig &c, PoolShape &d, std::string &why) {
    auto no = [&](const char *m) { why = std::string("kv_pool: ") + m; return false; };
    if (c.struct_size != sizeof(KronosCudaKvPoolConfig)) return no("struct_size does not match this library");
    if (c.kv_heads < 1 || c.kv_heads > 256) return no("1..256 kv heads");
    if (c.head_dim != 64 && c.head_dim != 128) return no("head_dim must be 64 or 128");
    if (c.kv_bits != 8 && c.kv_bits != 4) return no("kv_bits must be 8 or 4");
    if (c.page_tokens != 16 && c.page_tokens != 32 && c.page_tokens != 64 && c.page_tokens != 128) return no("page_tokens must be 16, 32, 64 or 128");
    if (c.num_pages < 1 || c.num_pages > 0x7fffffffu) return no("1..2^31-1 pages");
    if (c.flags & ~KRONOS_CUDA_POOL_BLOCK_KEYS) return no("unknown flag");
    d.kv_heads = c.kv_heads;
    d.head_dim = c.head_dim;
    d.bits = c.kv_bits;
    d.page_shift = c.page_tokens == 16 ? 4 : c.page_tokens == 32 ? 5 : c.page_tokens == 64 ? 6 : 7;
    d.num_pages = c.num_pages;
    d.block_keys = (c.flags & KRONOS_CUDA_POOL_BLOCK_KEYS) != 0;
    return true;
}

bool pool_rows(const PoolShape &d, uint32_t type, uint32_t heads, size_t n_tok, const KronosCudaRows &r, const char *name, bool written, RowsArg &out, std::string &why) {
    auto no = [&](const char *m) { why = std::string("kv_pool: ") + name + m; return false; };
    if (type != KRONOS_CUDA_TYPE_F32 && type != KRONOS_CUDA_TYPE_BF16 && type != KRONOS_CUDA_TYPE_F16) return no(": unknown type");
    if (r.data == nullptr && n_tok > 0) return no(" is NULL");          // of no token every address will do: empty buffers have none
    const uint64_t size = type == KRONOS_CUDA_TYPE_F32 ? 4 : 2;
    const uint64_t hs = r.head_stride != 0 ? r.head_stride : d.head_dim, ts = r.token_stride != 0 ? r.token_stride : heads * hs;
    if (hs >> 40 || ts >> 40) return no(": stride too large");
    if (reinterpret_cast<uint64_t>(r.data) % size != 0) return no(": not aligned to its elements");
    // rows that are written lie apart: tokens outermost, or heads
    if (written && (hs < d.head_dim || ts < d.head_dim || !(ts >= (heads - 1) * hs + d.head_dim || (n_tok >> 24 == 0 && hs >= (n_tok - 1) * ts + d.head_dim))) && n_tok > 0)
        return no(": rows overlap");
    out.p = r.data;
    out.token_stride = ts;
    out.head_stride = hs;
    out.type = type;
    out.wide = (reinterpret_cast<uint64_t>(r.data) | ts * size | hs * size) % 16 == 0;
    return true;
}

// Sizes that no attention call takes: the message, or null.
static const char *size_refusal(const PoolShape &d, uint32_t heads, uint32_t n_tok, uint32_t prefix_len) {
    if (heads < d.kv_heads || heads % d.kv_heads != 0 || heads / d.kv_heads > 256) return "heads must be 1..256 times the kv heads";
    if (n_tok > (1u << 20) || (uint64_t)n_tok * heads > 0x7fffffffu) return "too many tokens";
    if (prefix_len > 0x7fffffffu) return "prefix too long";
    if (((uint64_t)n_tok * heads / 64 + d.kv_heads) * (prefix_len / 64 + 1) >= MOST_TILES) return "prefix too long for so many tokens";
    return nullptr;
}
size_t pool_workspace(const PoolShape &d, uint32_t heads, uint32_t n_tok, uint32_t prefix_len, uint32_t sm_count) {
    return size_refusal(d, heads, n_tok, prefix_len) != nullptr ? 0 : pool_work_bytes(d, heads, n_tok, prefix_len, sm_count);
}

bool pool_attention(const PoolShape &d, const KronosCudaPoolAttention &c, int what, uint32_t sm_count, PoolAttnArgs &a, std::string &why) {
    auto no = [&](const char *m) { why = std::string("kv_pool: ") + m; return false; };
    const bool selects = what == POOL_SELECT, chosen = what != POOL_ATTEND;
    if (c.struct_size != sizeof(KronosCudaPoolAttention)) return no("struct_size does not match this library");
    if (const char *m = size_refusal(d, c.heads, c.n_tok, c.prefix_len)) return no(m);
    const bool some = c.n_tok > 0;
    if (some && (!c.lens || !c.pages)) return no("NULL table or lengths");
    if (c.pages_stride < 1 || c.pages_stride > (1u << 27)) return no("pages_stride must be 1..2^27");
    if (c.prefix_len > 0 && (chosen || (some && !c.prefix_pages))) return no(chosen ? "chosen pages do not go with a prefix" : "prefix without its pages");
    if (!(c.scale >= 0.0f) || c.scale > 1e30f) return no("scale must be a number from 0 on (0: 1 / sqrt(head_dim))");
    if (chosen) {
        if (some && !c.chosen) return no("chosen is NULL");
        if (c.top < 1 || c.top > KRONOS_CUDA_POOL_MAX_CHOSEN) return no("top must be 1..32768");
    } else if (c.chosen || c.top) {
        return no("attend takes no chosen pages (kronos_cuda_kv_pool_attend_chosen_dev)");
    }
    if (selects) {
        if (!d.block_keys) return no("select needs a pool with block keys");
        if (c.local < 1 || c.sinks > c.top || c.local > c.top - c.sinks) return no("select keeps at least the last page: local >= 1, sinks + local <= top");
        if (c.pages_stride > KRONOS_CUDA_POOL_MAX_CHOSEN) return no("select looks through at most 32768 pages of a sequence");
    }
    a.pool.d = d;
    if (!pool_rows(d, c.row_type, c.heads, c.n_tok, c.q, "q", false, a.q, why)) return false;
    if (!selects && !pool_rows(d, c.row_type, c.heads, c.n_tok, c.out, "out", true, a.out, why)) return false;
    a.n_tok = c.n_tok;
    a.heads = c.heads;
    a.lens = c.lens;
    a.seq = c.seq;
    a.pages = c.pages;
    a.pages_stride = c.pages_stride;
    a.prefix_pages = c.prefix_pages;
    a.prefix_len = c.prefix_len;
    a.scale = c.scale != 0.0f ? c.scale : d.head_dim == 64 ? 0.125f : 0.08838834764831845f;
    a.chosen = chosen ? c.chosen : nullptr;
    a.top = c.top;
    a.sinks = c.sinks;
    a.local = c.local;
    a.sm_count = sm_count;
    a.work = static_cast<uint8_t *>(c.workspace);
    if (!selects) {
        const size_t need = pool_work_bytes(d, c.heads, c.n_tok, c.prefix_len, sm_count);
        if (need > 0 && (!c.workspace || reinterpret_cast<uint64_t>(c.workspace) % 16 != 0)) return no("the workspace must be a 16-byte aligned device buffer");
        if (c.workspace_bytes < need) return no("workspace too small (kronos_cuda_kv_pool_workspace)");
    }
    return true;
}

// The same checks by a C interface, for hosts without a device: the message, or null.
const char *pool_refusal(const KronosCudaKvPoolConfig *config, const KronosCudaPoolAttention *c, int32_t what) {
    static thread_local std::string why;
    PoolShape d{};
    PoolAttnArgs a{};
    why.clear();
    if (!pool_shape(*config, d, why)) return why.c_str();
    if (c != nullptr && !pool_attention(d, *c, what, 148, a, why)) return why.c_str();
    return nullptr;
}

}  // namespace k2t

using namespace k2t;

namespace {

bool usable(KronosCudaContext *ctx, const KronosCudaKvPool *pool) {
    if (!pool) return fail(ctx, "kv_pool: pool is NULL");
    if (pool->device != ctx->device) return fail(ctx, "kv_pool: the pool lives on another device");
    return make_current(ctx);
}

int32_t move_rows(KronosCudaContext *ctx, KronosCudaKvPool *pool, uint32_t type, const KronosCudaRows *k, const KronosCudaRows *v, const int64_t *slots, size_t n_tok, bool load) {
    if (!ctx) return -1;
    ctx->err.clear();
    if (!usable(ctx, pool)) return -1;
    PoolStoreArgs a{};
    std::string why;
    if (!k || !v) return fail(ctx, "kv_pool: NULL rows"), -1;
    const PoolShape &d = pool->view.d;
    if (n_tok > (1u << 24) || n_tok * 2 * d.kv_heads >= 1ull << 31) return fail(ctx, "kv_pool: too many tokens"), -1;
    if (!pool_rows(d, type, d.kv_heads, n_tok, *k, "k", load, a.k, why) || !pool_rows(d, type, d.kv_heads, n_tok, *v, "v", load, a.v, why)) return fail(ctx, why), -1;
    if (n_tok == 0) return 0;
    if (!slots) return fail(ctx, "kv_pool: NULL slots"), -1;
    a.pool = pool->view;
    a.pool.err = ctx->d_err;
    a.slots = slots;
    a.n_tok = (uint32_t)n_tok;
    a.sm_count = pool->sm_count;
    uint32_t launched = 0;
    const cudaError_t e = load ? launch_pool_load(ctx->stream, a, &launched) : launch_pool_store(ctx->stream, a, &launched);
    ctx->launches += launched;
    return cuda_ok(ctx, e, load ? "kv_pool load" : "kv_pool store") ? 0 : -1;
}

int32_t attention(KronosCudaContext *ctx, KronosCudaKvPool *pool, const KronosCudaPoolAttention *c, int what) {
    if (!ctx) return -1;
    ctx->err.clear();
    if (!usable(ctx, pool)) return -1;
    if (!c) return fail(ctx, "kv_pool: arguments are NULL"), -1;
    PoolAttnArgs a{};
    std::string why;
    if (!pool_attention(pool->view.d, *c, what, pool->sm_count, a, why)) return fail(ctx, why), -1;
    if (c->n_tok == 0) return 0;
    a.pool = pool->view;
    a.pool.err = ctx->d_err;
    uint32_t launched = 0;
    const cudaError_t e = what == POOL_SELECT ? launch_pool_select(ctx->stream, a, &launched) : launch_pool_attend(ctx->stream, a, &launched);
    ctx->launches += launched;
    return cuda_ok(ctx, e, what == POOL_SELECT ? "kv_pool select" : "kv_pool attend") ? 0 : -1;
}

}  // namespace

extern "C" {

KronosCudaKvPool *kronos_cuda_kv_pool_create(KronosCudaContext *ctx, const KronosCudaKvPoolConfig *config) {
    if (!ctx) return nullptr;
    ctx->err.clear();
    if (!config) { fail(ctx, "kv_pool: config is NULL"); return nullptr; }
    PoolShape d{};
    std::string why;
    if (!pool_shape(*config, d, why)) { fail(ctx, why); return nullptr; }
    if (!make_current(ctx)) return nullptr;
    KronosCudaKvPool *pool = new (std::nothrow) KronosCudaKvPool();
    if (!pool) { fail(ctx, "kv_pool: out of host memory"); return nullptr; }
    pool->device = ctx->device;
    pool->sm_count = (uint32_t)ctx->sm_count;
    pool->view.d = d;
    for (uint32_t i = 0; i < 128; ++i) pool->view.signs[i / 32] |= sign_bit(i / 64, i % 64) << (i % 32);
    const size_t rows = (d.rows_bytes() + 255) & ~(size_t)255, keys = (d.key_bytes() + 255) & ~(size_t)255;
    pool->bytes = rows + keys + d.key_scale_bytes();
    uint8_t *base = nullptr;
    const cudaError_t e = cudaMalloc(reinterpret_cast<void **>(&base), pool->bytes);
    if (e == cudaErrorMemoryAllocation) cudaGetLastError();
    if (!cuda_ok(ctx, e, "cudaMalloc(kv_pool)")) { delete pool; return nullptr; }
    // rows nobody has written are rows of zeros: codes 0 (8-bit ones are stored with their sign bit flipped), scales 0
    const size_t block = d.block_bytes(), scales = 2 * d.scale_bytes(), blocks = d.rows_bytes() / block;
    if (!cuda_ok(ctx, cudaMemsetAsync(base, 0x80, rows, ctx->stream), "clear kv_pool") ||
        !cuda_ok(ctx, cudaMemset2DAsync(base + block - scales, block, 0, scales, blocks, ctx->stream), "clear kv_pool") ||
        !cuda_ok(ctx, cudaMemsetAsync(base + rows, 0, pool->bytes - rows, ctx->stream), "clear kv_pool") ||
        !cuda_ok(ctx, cudaStreamSynchronize(ctx->stream), "clear kv_pool")) {
        cudaFree(base);
        delete pool;
        return nullptr;
    }
    pool->view.rows = base;
    pool->view.block_keys = d.block_keys ? reinterpret_cast<int8_t *>(base + rows) : nullptr;
    pool->view.block_key_scales = d.block_keys ? reinterpret_cast<float *>(base + rows + keys) : nullptr;
    return pool;
}

void kronos_cuda_kv_pool_free(KronosCudaContext *ctx, KronosCudaKvPool *pool) {
    if (!pool) return;
    cudaSetDevice(pool->device);
    if (ctx && ctx->device == pool->device) cudaStreamSynchronize(ctx->stream);
    cudaFree(pool->view.rows);
    delete pool;
}

size_t kronos_cuda_kv_pool_bytes(const KronosCudaKvPool *pool) { return pool ? pool->bytes : 0; }

int32_t kronos_cuda_kv_pool_store_dev(KronosCudaContext *ctx, KronosCudaKvPool *pool, uint32_t type, const KronosCudaRows *d_k, const KronosCudaRows *d_v,
                                      const int64_t *d_slots, size_t n_tok) {
    return move_rows(ctx, pool, type, d_k, d_v, d_slots, n_tok, false);
}
int32_t kronos_cuda_kv_pool_load_dev(KronosCudaContext *ctx, KronosCudaKvPool *pool, uint32_t type, const KronosCudaRows *d_k, const KronosCudaRows *d_v,
                                     const int64_t *d_slots, size_t n_tok) {
    return move_rows(ctx, pool, type, d_k, d_v, d_slots, n_tok, true);
}

size_t kronos_cuda_kv_pool_workspace(const KronosCudaKvPool *pool, uint32_t heads, uint32_t n_tok, uint32_t prefix_len) {
    return pool ? pool_workspace(pool->view.d, heads, n_tok, prefix_len, pool->sm_count) : 0;
}

int32_t kronos_cuda_kv_pool_attend_dev(KronosCudaContext *ctx, KronosCudaKvPool *pool, const KronosCudaPoolAttention *args) { return attention(ctx, pool, args, POOL_ATTEND); }
int32_t kronos_cuda_kv_pool_attend_chosen_dev(KronosCudaContext *ctx, KronosCudaKvPool *pool, const KronosCudaPoolAttention *args) { return attention(ctx, pool, args, POOL_CHOSEN); }
int32_t kronos_cuda_kv_pool_select_dev(KronosCudaContext *ctx, KronosCudaKvPool *pool, const KronosCudaPoolAttention *args) { return attention(ctx, pool, args, POOL_SELECT); }

}  // extern "C"
