"""The shared pool of cached keys and values on the device, against tests/kv_pool_ref.py: rows bit for bit, choices of pages exactly, attention
within the bound that the roundings of its operands allow."""
import numpy as np
import pytest

import kv_pool_ref as ref

pytestmark = pytest.mark.gpu

HALF = {"f32": 2.0 ** -21, "bf16": 2.0 ** -11, "f16": 2.0 ** -11}        # operands of the products: two halves, or one
OUT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


@pytest.fixture(scope="module")
def ctx():
    import torch

    import kronos_2t_b200 as k2
    c = k2.Context(0)
    c.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    yield c
    c.close()


def torch_type(dtype):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]


def device(x, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(torch_type(dtype))


def rounded(x, dtype):
    """fp32 values as they are in `dtype`."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch_type(dtype)).float().numpy()


class Cache:
    """A pool and the same rows in numpy: sequences of given lengths in pages dealt out at random, garbage behind the last row of each."""

    def __init__(self, ctx, lens, kh, d, bits, page, dtype, prefix=0, seed=0, block_keys=False, room=0):
        from kronos_2t_b200 import KvPool
        rng = self.rng = np.random.default_rng(seed)
        self.ctx, self.kh, self.d, self.bits, self.page, self.dtype, self.prefix = ctx, kh, d, bits, page, dtype, prefix
        counts = [-(-n // page) for n in lens]
        far = -(-prefix // page)
        total = far + sum(counts) + 3
        self.pool = KvPool(ctx, kh, d, bits, page, total, block_keys=block_keys)
        order = rng.permutation(total)
        self.prefix_pages, at = order[:far].astype(np.int32), far
        width = max([1] + counts) + room
        self.table = rng.choice(np.array([-7, 1 << 30, 0], np.int32), (len(lens), width))       # behind the last page: anything
        for b, c in enumerate(counts):
            self.table[b, :c] = order[at:at + c]
            at += c
        # every slot holds rows that are not finite before the sequences' own are written
        every = np.arange(total * page)
        self.store(every, np.full((every.size, kh, d), np.nan, np.float32), np.full((every.size, kh, d), np.nan, np.float32))
        self.far = self.fill(prefix, self.prefix_pages)
        self.own = [self.fill(n, self.table[b]) for b, n in enumerate(lens)]

    def fill(self, n, pages):
        rng, (kh, d) = self.rng, (self.kh, self.d)
        k = rounded(rng.standard_normal((n, kh, d)) * (1 + 4 * (rng.random((kh, d)) > 0.95)), self.dtype)
        v = rounded(rng.standard_normal((n, kh, d)), self.dtype)
        at = np.arange(n)
        if n:
            self.store(pages[at // self.page].astype(np.int64) * self.page + at % self.page, k, v)
        return ref.stored(k, self.bits).reshape(n, kh, d), ref.stored(v, self.bits).reshape(n, kh, d)

    def store(self, slots, k, v):
        dk, dv, ds = device(k, self.dtype), device(v, self.dtype), device(slots.astype(np.int64))
        self.pool.store_dev(self.dtype, dk.data_ptr(), dv.data_ptr(), ds.data_ptr(), len(slots))
        self.ctx.synchronize()

    def queries(self, n, heads):
        return rounded(self.rng.standard_normal((n, heads, self.d)) * 1.5, self.dtype)

    def attend(self, q, lens, seq=None, chosen=None, scale=0.0, table=None):
        import torch
        n, heads, _ = q.shape
        dq, dl = device(q, self.dtype), device(np.asarray(lens, np.int32))
        dt = device(self.table if table is None else table)
        ds = None if seq is None else device(np.asarray(seq, np.int32))
        out = torch.full(q.shape, float("nan"), device="cuda", dtype=torch_type(self.dtype))
        size = self.pool.workspace_bytes(heads, n, self.prefix if chosen is None else 0)
        work = torch.full((size + 16,), 255, dtype=torch.uint8, device="cuda")
        args = dict(dtype=self.dtype, heads=heads, n_tok=n, d_q=dq.data_ptr(), d_lens=dl.data_ptr(), d_pages=dt.data_ptr(), pages_stride=dt.shape[1],
                    d_seq=None if ds is None else ds.data_ptr(), workspace=(work.data_ptr(), size), d_out=out.data_ptr(), scale=scale)
        if chosen is None:
            far = device(self.prefix_pages if self.prefix else np.zeros(1, np.int32))
            self.pool.attend_dev(**args, d_prefix_pages=far.data_ptr(), prefix_len=self.prefix)
        else:
            dc = device(np.asarray(chosen, np.int32))
            self.pool.attend_chosen_dev(**args, top=dc.shape[2], d_chosen=dc.data_ptr())
        torch.cuda.synchronize()
        return out.float().cpu().numpy()

    def select(self, q, lens, top, sinks, local, seq=None):
        import torch
        n, heads, _ = q.shape
        dq, dl, dt = device(q, self.dtype), device(np.asarray(lens, np.int32)), device(self.table)
        ds = None if seq is None else device(np.asarray(seq, np.int32))
        out = torch.full((n, self.kh, top), 77, dtype=torch.int32, device="cuda")
        self.pool.select_dev(self.dtype, heads, n, dq.data_ptr(), dl.data_ptr(), dt.data_ptr(), dt.shape[1], top, out.data_ptr(), sinks=sinks, local=local,
                             d_seq=None if ds is None else ds.data_ptr())
        torch.cuda.synchronize()
        return out.cpu().numpy()

    def check(self, got, q, lens, seq=None, scale=None, rows_of=None):
        """Every token's output within the bound; rows_of(t, kv head) picks rows of the sequence (all in sight otherwise)."""
        d, heads = self.d, q.shape[1]
        scale = d ** -0.5 if scale is None else scale
        assert np.isfinite(got).all()
        for t in range(q.shape[0]):
            b = t if seq is None else seq[t]
            n = 0 if b < 0 else max(0, lens[t])
            for h in range(self.kh):
                mine = slice(h * heads // self.kh, (h + 1) * heads // self.kh)
                rows = np.arange(n) if rows_of is None else rows_of(t, h)
                pick = (lambda x: x[rows, h:h + 1]) if n else (lambda x: x[:0, h:h + 1])
                k, v = (np.concatenate((self.far[i][:, h:h + 1], pick(self.own[max(b, 0)][i]))) for i in range(2))
                want, bound = ref.attend(q[t, mine], k, v, scale, HALF[self.dtype])
                off = np.linalg.norm((got[t, mine] - want).reshape(-1, d // 64, 64), axis=-1)
                allowed = bound * (1 + OUT[self.dtype]) + OUT[self.dtype] * np.linalg.norm(want.reshape(-1, d // 64, 64), axis=-1) + 1e-7
                if self.dtype == "f16":
                    allowed += 8 * 2.0 ** -25          # below the smallest ordinary half: half a step of 2^-24 in each of 64 values
                assert (off <= allowed).all(), (t, h, off.max(), allowed[off > allowed], off[off > allowed])


SHAPES = [(128, 8), (128, 4), (64, 8), (64, 4)]


# ------------------------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("d,bits", SHAPES)
@pytest.mark.parametrize("dtype,page,kh", [("f32", 16, 1), ("bf16", 64, 3), ("f16", 128, 8), ("bf16", 32, 5)])
def test_rows_come_back_as_their_definition_says(ctx, d, bits, dtype, page, kh):
    import torch

    from kronos_2t_b200 import KvPool
    rng = np.random.default_rng(d + bits)
    n, pages = 37, 9
    x = [rounded(rng.standard_normal((n, kh, d)) * 10.0 ** rng.integers(-3, 3, (n, kh, 1)), dtype) for _ in range(2)]
    for i in range(2):
        x[i][3] = 0
        x[i][4] = rounded(np.full((kh, d), 1e-9, np.float32), dtype)        # below what 8-bit rows keep
        x[i][5, 0, 7] = np.inf
        x[i][6, kh - 1, d - 1] = np.nan
    slots = rng.permutation(pages * page)[:n].astype(np.int64)
    slots[[8, 20]] = -1
    pool = KvPool(ctx, kh, d, bits, page, pages)
    dx, ds = [device(a, dtype) for a in x], device(slots)
    pool.store_dev(dtype, dx[0].data_ptr(), dx[1].data_ptr(), ds.data_ptr(), n)
    for out_type in ("f32", "bf16", "f16"):
        out = [torch.full((n, kh, d), 5.0, device="cuda", dtype=torch_type(out_type)) for _ in range(2)]
        pool.load_dev(out_type, ds.data_ptr(), n, out[0].data_ptr(), out[1].data_ptr())
        ctx.synchronize()
        for i in range(2):
            want = rounded(ref.read_back(x[i], bits), out_type)
            want[[8, 20]] = 5.0
            assert np.isnan(want[5, 0]).all() and np.isnan(want[6, kh - 1]).all() and np.isfinite(want[7]).all()
            assert np.array_equal(out[i].float().cpu().numpy(), want, equal_nan=True)
    # a slot that nobody wrote holds zeros
    free = np.setdiff1d(np.arange(pages * page), slots)[:1].astype(np.int64)
    df, out = device(free), [torch.full((1, kh, d), 5.0, device="cuda") for _ in range(2)]
    pool.load_dev("f32", df.data_ptr(), 1, out[0].data_ptr(), out[1].data_ptr())
    ctx.synchronize()
    assert not any(o.any() for o in out)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("token,head,offset", [(1000, 128, 0), (128, 40 * 128 + 8, 0), (531, 131, 1), (4 * 128 + 4, 128, 3)])
def test_rows_with_strides(ctx, dtype, token, head, offset):
    """Rows inside a wider buffer, heads outermost, and at addresses that allow no wide access."""
    import torch

    from kronos_2t_b200 import KvPool
    n, kh, d, rng = 40, 4, 128, np.random.default_rng(token)
    flat = rounded(rng.standard_normal(max(n * token, kh * head) + token + head + 64), dtype)
    at = offset + np.arange(n)[:, None, None] * token + np.arange(kh)[None, :, None] * head + np.arange(d)
    pool, buf, slots = KvPool(ctx, kh, d, 8, 16, 4), device(flat, dtype), device(np.arange(n, dtype=np.int64))
    rows = (buf.data_ptr() + offset * buf.element_size(), token, head)
    pool.store_dev(dtype, rows, rows, slots.data_ptr(), n)
    out = [torch.full((flat.size,), 3.0, device="cuda", dtype=torch_type(dtype)) for _ in range(2)]
    back = [(o.data_ptr() + offset * o.element_size(), token, head) for o in out]
    pool.load_dev(dtype, slots.data_ptr(), n, back[0], back[1])
    ctx.synchronize()
    want = np.full(flat.size, 3.0, np.float32)
    want[at] = rounded(ref.read_back(flat[at], 8), dtype)
    for o in out:
        assert np.array_equal(o.float().cpu().numpy(), want)


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("d,bits", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kh,heads,page", [(2, 14, 64), (3, 3, 16), (1, 20, 128), (4, 64, 32)])
def test_attention_of_ragged_sequences(ctx, d, bits, dtype, kh, heads, page):
    lens = [0, 1, 15, 16, 17, 64, 65, 300, 1000][:9 if kh < 4 else 7]
    c = Cache(ctx, lens, kh, d, bits, page, dtype, seed=heads, room=2)
    q = c.queries(len(lens), heads)
    got = c.attend(q, lens)
    assert not got[0].any()
    c.check(got, q, lens)


@pytest.mark.parametrize("d,bits", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("prefix,kh,heads,page,seqs,new", [(1, 2, 2, 16, 1, 1), (33, 3, 9, 16, 3, 1), (500, 2, 14, 64, 9, 1), (129, 1, 8, 128, 5, 4), (1000, 2, 32, 32, 20, 1)])
def test_attention_behind_a_shared_prefix(ctx, d, bits, dtype, prefix, kh, heads, page, seqs, new):
    """Also several new tokens of a sequence, each seeing one more of its rows; a sequence without rows; a padding token."""
    rng = np.random.default_rng(seqs)
    ends = rng.integers(new, 90, seqs)
    if new == 1 and seqs > 1:
        ends[1] = 0
    c = Cache(ctx, ends, kh, d, bits, page, dtype, prefix=prefix, seed=prefix)
    seq = np.repeat(np.arange(seqs), new)
    lens = (ends[:, None] - new + 1 + np.arange(new)).reshape(-1)
    if new == 1:
        lens = ends.copy()
    if seqs > 2:
        seq[2] = -1
    q = c.queries(seqs * new, heads)
    got = c.attend(q, lens, seq)
    c.check(got, q, lens, seq)


@pytest.mark.parametrize("d,bits", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("prefix,kh,heads,seqs", [(3001, 8, 64, 40), (2500, 5, 5, 100), (9000, 1, 6, 45), (20000, 2, 2, 17)])
def test_a_prefix_over_many_rows(ctx, d, bits, dtype, prefix, kh, heads, seqs):
    """Rows of several tiles, parts that begin and end inside an item, and items of one tile of rows."""
    rng = np.random.default_rng(seqs)
    ends = rng.integers(0, 40, seqs)
    c = Cache(ctx, ends, kh, d, bits, 64, dtype, prefix=prefix, seed=prefix)
    q = c.queries(seqs, heads)
    got = c.attend(q, ends)
    assert np.array_equal(got, c.attend(q, ends))
    pick = rng.permutation(seqs)[:6]
    c.check(got[pick], q[pick], ends[pick], pick)


@pytest.mark.parametrize("prefix", [0, 70])
def test_many_short_tokens(ctx, prefix):
    """More items than warps: one warp each."""
    rng = np.random.default_rng(3)
    ends = rng.integers(0, 40, 50)
    c = Cache(ctx, ends, 8, 64, 8, 16, "bf16", prefix=prefix)
    seq = rng.integers(0, 50, 1100)
    lens = np.minimum(rng.integers(0, 41, 1100), ends[seq])
    q = c.queries(1100, 8)
    got = c.attend(q, lens, seq)
    pick = rng.permutation(1100)[:60]
    c.check(got[pick], q[pick], lens[pick], seq[pick])


@pytest.mark.parametrize("bits", [8, 4])
def test_one_long_sequence(ctx, bits):
    """One token's rows over all warps; keys that stand out first, in the middle and last."""
    n = 20011
    c = Cache(ctx, [n], 2, 128, bits, 64, "f32", seed=bits)
    q = c.queries(1, 8)
    c.check(c.attend(q, [n]), q, [n])
    for at in (0, 10007, n - 1):
        k = np.repeat(q[0].reshape(2, 4, 128).sum(1)[None], 1, 0).astype(np.float32) * 2
        v = c.rng.standard_normal((1, 2, 128)).astype(np.float32)
        c.store(np.array([c.table[0][at // 64] * 64 + at % 64]), k, v)
        for i, x in enumerate((k, v)):
            c.own[0][i][at] = ref.stored(x, bits)[0]
    c.check(c.attend(q, [n]), q, [n])


def test_values_and_scores_of_all_sizes(ctx):
    """Rows whose scales lie far apart, rows of zeros, very large and very small queries."""
    rng = np.random.default_rng(1)
    c = Cache(ctx, [200], 1, 128, 8, 64, "f32")
    k, v = (rng.standard_normal((200, 1, 128)).astype(np.float32) for _ in range(2))
    v *= 10.0 ** rng.integers(-6, 7, (200, 1, 1))
    v[::7] = 0
    k[::11] = 0
    c.store(c.table[0][np.arange(200) // 64].astype(np.int64) * 64 + np.arange(200) % 64, k, v)
    c.own[0] = ref.stored(k, 8), ref.stored(v, 8)
    q = c.queries(1, 6)
    for size in (1e-30, 1e-3, 1.0, 3.0):
        c.check(c.attend((q * np.float32(size)), [200]), (q * np.float32(size)).astype(np.float32), [200])
    got = c.attend(np.zeros_like(q), [200])           # every row alike
    c.check(got, np.zeros_like(q), [200])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_scale_strides_and_heads_outermost(ctx, dtype):
    import torch
    lens, heads, d = [40, 3, 100], 8, 64
    c = Cache(ctx, lens, 2, d, 8, 16, dtype)
    q = c.queries(3, heads)
    c.check(c.attend(q, lens, scale=0.3), q, lens, scale=0.3)
    straight = c.attend(q, lens)
    wide = torch.full((heads, 3, d + 3), 2.0, device="cuda", dtype=torch_type(dtype))
    wide[:, :, 1:d + 1] = device(q, dtype).transpose(0, 1)
    out, dl, dt = torch.full_like(wide, 9.0), device(np.array(lens, np.int32)), device(c.table)
    work = torch.empty(c.pool.workspace_bytes(heads, 3), dtype=torch.uint8, device="cuda")
    size = wide.element_size()
    c.pool.attend_dev(dtype, heads, 3, (wide.data_ptr() + size, d + 3, 3 * (d + 3)), dl.data_ptr(), dt.data_ptr(), dt.shape[1],
                      (out.data_ptr() + size, d + 3, 3 * (d + 3)), (work.data_ptr(), work.numel()))
    ctx.synchronize()
    got = out.float().cpu().numpy()
    assert np.array_equal(got[:, :, 1:d + 1].transpose(1, 0, 2), straight)
    assert (got[:, :, 0] == 9).all() and (got[:, :, d + 1:] == 9).all()


def test_a_row_that_is_not_finite_reaches_those_that_see_it(ctx):
    lens = [30, 30, 64]
    c = Cache(ctx, lens, 2, 64, 8, 16, "bf16")
    q = c.queries(3, 4)
    bad = np.zeros((1, 2, 64), np.float32)
    bad[0, 1, 5] = np.inf
    good = rounded(np.ones((1, 2, 64)), "bf16")
    c.store(np.array([c.table[1][1] * 16 + 4]), bad, good)                       # row 20 of sequence 1: head 1's key
    got = c.attend(q, lens)
    assert np.isnan(got[1, 2:]).all() and np.isfinite(np.delete(got, 1, 0)).all() and np.isfinite(got[1, :2]).all()
    assert np.isfinite(c.attend(q, [30, 20, 64])).all()                           # out of sight
    q[0, 3] = np.nan                                                              # a query of its own
    got = c.attend(q, [30, 20, 64])
    assert np.isnan(got[0, 3]).all() and np.isfinite(got[0, :3]).all() and np.isfinite(got[1:]).all()


# ------------------------------------------------------------------------------------------------ chosen pages
def keys_of(c, b):
    whole = c.own[b][0].shape[0] // c.page
    got = [ref.block_key(c.own[b][0][i * c.page:(i + 1) * c.page]) for i in range(whole)]
    return np.stack([g[0] for g in got]), np.stack([g[1] for g in got])


@pytest.mark.parametrize("d,bits", SHAPES)
@pytest.mark.parametrize("dtype,kh,heads,page", [("bf16", 2, 14, 16), ("f32", 3, 3, 32), ("f16", 1, 20, 128)])
def test_choice_and_attention_over_it(ctx, d, bits, dtype, kh, heads, page):
    lens = [1, page, 5 * page, 6 * page + 1, 40 * page - 3, 700]
    c = Cache(ctx, lens, kh, d, bits, page, dtype, block_keys=True, seed=d + bits)
    q = c.queries(len(lens), heads)
    for top, sinks, local in ((6, 1, 2), (1, 0, 1), (5, 2, 3), (9, 0, 1), (50, 3, 1)):
        got = c.select(q, lens, top, sinks, local)
        for t, n in enumerate(lens):
            keys, scales = keys_of(c, t) if n >= page else (np.zeros((0, kh, d)), np.zeros((0, kh)))
            assert np.array_equal(got[t], ref.select(q[t], keys, scales, -(-n // page), top, sinks, local)), (t, top)
        out = c.attend(q, lens, chosen=got)

        def rows_of(t, h):
            at = (got[t, h][got[t, h] >= 0][:, None] * page + np.arange(page)).reshape(-1)
            return at[at < lens[t]]
        c.check(out, q, lens, rows_of=rows_of)


def test_choice_among_equals_and_pages_that_are_not_finite(ctx):
    """The lowest index first; a page with a key that is not finite behind all others; a query of zeros scores all alike."""
    page, n = 16, 20 * 16
    c = Cache(ctx, [n], 1, 64, 8, page, "f32", block_keys=True)
    one = c.rng.standard_normal((page, 1, 64)).astype(np.float32)
    k = np.concatenate([one * (2 if i in (4, 9, 17) else 1) for i in range(20)])
    k[3 * page, 0, 0] = np.nan
    c.store(c.table[0][np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page, k, k)
    q = (k[4 * page:5 * page].sum(0) / 4)[None].astype(np.float32)
    assert c.select(q, [n], 5, 0, 1)[0, 0].tolist() == [0, 4, 9, 17, 19]
    assert c.select(q, [n], 4, 0, 1)[0, 0].tolist() == [4, 9, 17, 19]
    assert c.select(-q, [n], 5, 1, 1)[0, 0].tolist() == [0, 1, 2, 5, 19]
    assert c.select(q * 0, [n], 5, 0, 2)[0, 0].tolist() == [0, 1, 2, 18, 19]
    assert 3 not in c.select(q, [n], 19, 0, 1)[0, 0] and 3 not in c.select(-q, [n], 19, 0, 1)[0, 0]


@pytest.mark.parametrize("tokens,pages", [(700, 30), (3, 6000), (1, 2000)])
def test_choice_of_many_tokens_and_among_many_pages(ctx, tokens, pages):
    """More (token, kv head) pairs than the SMs hold, and more pages than threads."""
    page, n = 16, pages * 16 - 5
    c = Cache(ctx, [n], 1, 64, 8, page, "f32", block_keys=True)
    q, rng = c.queries(tokens, 2), np.random.default_rng(tokens)
    lens = np.maximum(1, n - rng.integers(0, n // 2, tokens))
    lens[0] = n
    keys, scales = keys_of(c, 0)
    got = c.select(q, lens, 24, 1, 2, seq=np.zeros(tokens, int))
    for t in range(0, tokens, max(1, tokens // 12)):
        assert np.array_equal(got[t], ref.select(q[t], keys, scales, -(-int(lens[t]) // page), 24, 1, 2)), t


def test_block_key_of_a_page_that_is_used_again(ctx):
    """The last row of a page makes its key from the rows that lie there then, also when they came in several calls."""
    page = 32
    c = Cache(ctx, [10 * page], 2, 128, 4, page, "bf16", block_keys=True)
    for first, n in ((64, 1), (65, 30), (95, 1), (200, 24)):             # page 2 in three calls; rows of page 6 up to its last one
        k, v = (rounded(c.rng.standard_normal((n, 2, 128)), "bf16") for _ in range(2))
        at = first + np.arange(n)
        c.store(c.table[0][at // page].astype(np.int64) * page + at % page, k, v)
        c.own[0][0][at], c.own[0][1][at] = ref.stored(k, 4), ref.stored(v, 4)
    q = c.queries(1, 8)
    keys, scales = keys_of(c, 0)
    for top in (2, 3, 4, 5, 6, 7, 8):
        assert np.array_equal(c.select(q, [10 * page], top, 0, 1)[0], ref.select(q[0], keys, scales, 10, top, 0, 1))


def test_choices_of_the_callers_own(ctx):
    """Any order, gaps, pages behind the last; a token that is left with none."""
    page, lens = 16, [100, 33]
    c = Cache(ctx, lens, 2, 128, 8, page, "f32")
    q = c.queries(2, 6)
    chosen = np.array([[[5, -1, 0, 6, 900], [-1, -1, -1, 3, -5]], [[2, 1, 0, 3, 4], [-1, -1, 7, -1, -1]]], np.int32)
    got = c.attend(q, lens, chosen=chosen)
    assert not got[1, 3:].any()

    def rows_of(t, h):
        pages = [p for p in chosen[t, h] if 0 <= p < -(-lens[t] // page)]
        at = (np.array(pages, int)[:, None] * page + np.arange(page)).reshape(-1)
        return at[at < lens[t]]
    want = got.copy()
    got[1, 3:] = 0
    c.check(got[:1], q[:1], lens[:1], rows_of=rows_of)
    for h in range(1):
        c.check(np.concatenate((want[:1], want[1:])), q, lens, rows_of=lambda t, h: rows_of(t, h))


# ------------------------------------------------------------------------------------------------ calls
def test_pages_and_slots_outside_the_pool_are_reported(ctx):
    """They are skipped: what is in sight stays right."""
    from kronos_2t_b200 import KronosCudaError
    page, lens = 16, [50, 60]
    c = Cache(ctx, lens, 1, 64, 8, page, "f32")
    q = c.queries(2, 4)
    good = c.attend(q, lens)
    for bad in (-1, 1 << 20):
        table = c.table.copy()
        table[1, 2] = bad
        got = c.attend(q, lens, table=table)
        with pytest.raises(KronosCudaError, match="outside the pool"):
            ctx.synchronize()
        ctx.synchronize()
        assert np.array_equal(got[0], good[0])
        c.check(got[1:], q[1:], lens[1:], seq=[1], rows_of=lambda t, h: np.array([i for i in range(60) if not 32 <= i < 48]))
    c.attend(q, [50, c.table.shape[1] * page + 1])                # longer than its table
    with pytest.raises(KronosCudaError, match="outside the pool"):
        ctx.synchronize()
    with pytest.raises(KronosCudaError, match="outside the pool"):
        c.store(np.array([1 << 40]), np.ones((1, 1, 64), np.float32), np.ones((1, 1, 64), np.float32))
    assert np.array_equal(c.attend(q, lens), good)
    ctx.synchronize()


@pytest.mark.parametrize("seqs,heads,prefix", [(1, 4, 400), (40, 4, 400), (25, 4, 5000), (90, 4, 1600)])
@pytest.mark.parametrize("d,bits", SHAPES)
def test_bad_pages_of_a_prefix_are_out_of_sight(ctx, seqs, heads, prefix, d, bits):
    """Few rows, one tile of them, two tiles; what is in sight stays right, and the call is reported."""
    from kronos_2t_b200 import KronosCudaError
    c = Cache(ctx, [5] * seqs, 1, d, bits, 16, "bf16", prefix=prefix)
    q = c.queries(seqs, heads)
    c.prefix_pages[[3, 11, 24]] = [-1, 1 << 20, 1 << 30]
    got = c.attend(q, [5] * seqs)
    with pytest.raises(KronosCudaError, match="outside the pool"):
        ctx.synchronize()
    keep = np.array([i for i in range(prefix) if i // 16 not in (3, 11, 24)])
    c.far = tuple(x[keep] for x in c.far)
    pick = np.arange(0, seqs, max(1, seqs // 3))
    c.check(got[pick], q[pick], [5] * len(pick), pick)
    ctx.synchronize()


@pytest.mark.parametrize("prefix", [600, 20000])
def test_the_same_call_gives_the_same_bits_also_captured_and_on_another_stream(ctx, prefix):
    """Two graphs with a workspace each, replayed in turn with new lengths and queries in place."""
    import torch
    lens = [900, 17, 300, 0]
    c = Cache(ctx, lens, 2, 128, 8, 64, "bf16", prefix=prefix)
    q = [c.queries(4, 16) for _ in range(2)]
    want = [c.attend(x, lens) for x in q]
    assert np.array_equal(want[0], c.attend(q[0], lens))
    stream = torch.cuda.Stream()
    dl, dt, far = device(np.array(lens, np.int32)), device(c.table), device(c.prefix_pages)
    dq, out = [device(x, "bf16") for x in q], [torch.zeros(4, 16, 128, dtype=torch.bfloat16, device="cuda") for _ in q]
    work = [torch.empty(c.pool.workspace_bytes(16, 4, prefix), dtype=torch.uint8, device="cuda") for _ in q]

    def call(i):
        c.pool.attend_dev("bf16", 16, 4, dq[i].data_ptr(), dl.data_ptr(), dt.data_ptr(), dt.shape[1], out[i].data_ptr(), (work[i].data_ptr(), work[i].numel()),
                          d_prefix_pages=far.data_ptr(), prefix_len=prefix)
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    try:
        graphs = [torch.cuda.CUDAGraph() for _ in q]
        for i, g in enumerate(graphs):
            with torch.cuda.graph(g, stream=stream):
                call(i)
        for _ in range(2):
            for o in out:
                o.zero_()
            torch.cuda.synchronize()
            for g in graphs:
                g.replay()
            torch.cuda.synchronize()
            for i in range(2):
                assert np.array_equal(out[i].float().cpu().numpy(), want[i])
        shorter = [100, 3, 300, 9]
        dl.copy_(device(np.array(shorter, np.int32)))
        dt[3, 0] = dt[0, 0]
        torch.cuda.synchronize()
        graphs[0].replay()
        torch.cuda.synchronize()
        c.own[3] = tuple(x[:9] for x in c.own[0])
        c.check(out[0].float().cpu().numpy(), q[0], shorter)
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)


def test_offsets_beyond_32_bits(ctx):
    """Rows behind the first 4 GB of a pool."""
    import torch

    from kronos_2t_b200 import KvPool
    page, kh, d, pages = 128, 8, 128, 17000
    pool = KvPool(ctx, kh, d, 8, page, pages, block_keys=True)
    assert pool.device_bytes > 1 << 32
    rng = np.random.default_rng(0)
    table = np.array([[pages - 1, 3, pages - 2]], np.int32)
    n = 300
    k, v = (rng.standard_normal((n, kh, d)).astype(np.float32) for _ in range(2))
    slots = table[0][np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page
    dk, dv, ds = device(k), device(v), device(slots)
    pool.store_dev("f32", dk.data_ptr(), dv.data_ptr(), ds.data_ptr(), n)
    back = [torch.empty(n, kh, d, device="cuda") for _ in range(2)]
    pool.load_dev("f32", ds.data_ptr(), n, back[0].data_ptr(), back[1].data_ptr())
    c = Cache(ctx, [1], kh, d, 8, page, "f32")
    c.pool, c.table, c.own = pool, table, [(ref.stored(k, 8), ref.stored(v, 8))]
    q = c.queries(1, 16)
    c.check(c.attend(q, [n]), q, [n])
    keys, scales = keys_of(c, 0)
    assert np.array_equal(c.select(q, [n], 2, 0, 1)[0], ref.select(q[0], keys, scales, 3, 2, 0, 1))
    ctx.synchronize()
    assert np.array_equal(back[0].cpu().numpy(), ref.read_back(k, 8)) and np.array_equal(back[1].cpu().numpy(), ref.read_back(v, 8))
    pool.free()


@pytest.mark.parametrize("bits", [8, 4])
def test_a_server_step_by_step(ctx, bits):
    """A prompt shared by all is written once; sequences of different lengths then grow token by token, each step stored, attended to behind
    the prefix, and attended to over chosen pages."""
    page, kh, heads, d, prefix, seqs = 16, 2, 8, 64, 75, 4
    start = [1, 14, 31, 60]
    c = Cache(ctx, start, kh, d, bits, page, "bf16", prefix=prefix, block_keys=True, room=3)
    free = [p for p in range(c.pool.num_pages) if p not in set(c.prefix_pages) | {p for b in range(seqs) for p in c.table[b, :-(-start[b] // page)]}]
    lens = list(start)
    for step in range(4):
        k, v = (rounded(c.rng.standard_normal((seqs, kh, d)), "bf16") for _ in range(2))
        slots = []
        for b in range(seqs):
            if lens[b] % page == 0:
                c.table[b, lens[b] // page] = free.pop()
            slots.append(int(c.table[b, lens[b] // page]) * page + lens[b] % page)
            c.own[b] = tuple(np.concatenate((old, ref.stored(new[b:b + 1], bits))) for old, new in zip(c.own[b], (k, v)))
            lens[b] += 1
        c.store(np.array(slots), k, v)
        q = c.queries(seqs, heads)
        c.check(c.attend(q, lens), q, lens)
        got = c.select(q, lens, 3, 1, 1)
        for b in range(seqs):
            keys, scales = keys_of(c, b) if lens[b] >= page else (np.zeros((0, kh, d)), np.zeros((0, kh)))
            assert np.array_equal(got[b], ref.select(q[b], keys, scales, -(-lens[b] // page), 3, 1, 1))
        out, far, c.far = c.attend(q, lens, chosen=got), c.far, tuple(x[:0] for x in c.far)
        c.check(out, q, lens, rows_of=lambda t, h: np.array([i for p in got[t, h] if p >= 0 for i in range(p * page, min(lens[t], (p + 1) * page))]))
        c.far = far


def test_calls_that_are_refused_leave_everything_as_it_is(ctx):
    import torch

    import kronos_2t_b200 as k2
    with pytest.raises(k2.KronosCudaError, match="head_dim"):
        k2.KvPool(ctx, 2, 96, 8, 16, 4)
    c = Cache(ctx, [20], 2, 64, 8, 16, "f32")
    q, out = device(c.queries(1, 4)), torch.full((1, 4, 64), 7.0, device="cuda")
    lens, table = device(np.array([20], np.int32)), device(c.table)
    work = torch.empty(64, dtype=torch.uint8, device="cuda")
    launches = ctx.launch_count
    with pytest.raises(k2.KronosCudaError, match="workspace too small"):
        c.pool.attend_dev("f32", 4, 1, q.data_ptr(), lens.data_ptr(), table.data_ptr(), table.shape[1], out.data_ptr(), (work.data_ptr(), 64))
    with pytest.raises(k2.KronosCudaError, match="block keys"):
        c.pool.select_dev("f32", 4, 1, q.data_ptr(), lens.data_ptr(), table.data_ptr(), table.shape[1], 2, work.data_ptr())
    with pytest.raises(k2.KronosCudaError, match="NULL slots"):
        c.pool.store_dev("f32", q.data_ptr(), q.data_ptr(), None, 1)
    c.pool.store_dev("f32", q.data_ptr(), q.data_ptr(), None, 0)
    assert ctx.launch_count == launches and (out == 7).all()
