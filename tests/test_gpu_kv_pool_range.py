"""The shared pool of cached keys and values on the device, at the ends of what its calls allow."""
import os
import subprocess
import sys

import numpy as np
import pytest

import kv_pool_ref as ref
from test_gpu_kv_pool import HALF, OUT, SHAPES, Cache, ctx, device, rounded, torch_type  # noqa: F401

pytestmark = pytest.mark.gpu

# ------------------------------------------------------------------------------------------------ wide tables
WIDE_TABLES = """
import sys
import numpy as np, torch
import kronos_2t_b200 as k2
d = int(sys.argv[1])
ctx = k2.Context(0)
ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
pool = k2.KvPool(ctx, 1, d, 8, 16, 64, block_keys=True)
rng = np.random.default_rng(0)
k = torch.from_numpy(rng.standard_normal((640, 1, d)).astype(np.float32)).cuda()
pool.store_dev("f32", k.data_ptr(), k.data_ptr(), torch.arange(640, device="cuda").data_ptr(), 640)
q = torch.from_numpy(rng.standard_normal((1, 1, d)).astype(np.float32)).cuda()
lens = torch.tensor([640], dtype=torch.int32, device="cuda")
want = None
for width in (40, 4096, 4097, 9788, 9789, 10240, 10892, 10893, 12287, 12288, 12289, 20000, 32768):
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, :40] = torch.arange(40)
    out = torch.full((1, 1, 9), 77, dtype=torch.int32, device="cuda")
    pool.select_dev("f32", 1, 1, q.data_ptr(), lens.data_ptr(), table.data_ptr(), width, 9, out.data_ptr(), sinks=1, local=1)
    ctx.synchronize()
    got = out.cpu().tolist()
    want = want or got
    assert got == want and got[0][0][0] == 0 and got[0][0][-1] == 39, (width, got, want)
print("widths agree")
"""

@pytest.mark.parametrize("d", [64, 128])
def test_choice_in_tables_of_every_width(d):
    """The table's width alone sizes the kernel's shared memory; in a process of its own, widths ascending, so that no wider call has gone before."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = subprocess.run([sys.executable, "-c", WIDE_TABLES, str(d)], cwd=root, capture_output=True, text=True, timeout=600)
    assert got.returncode == 0 and "widths agree" in got.stdout, got.stderr[-2000:]


# ------------------------------------------------------------------------------------------------ rows of zeros, scales far apart
def value_parts(v, bits):
    """Codes [rows][d] and the larger scale of each row of transformed value rows as they are stored."""
    if bits == 8:
        scale = np.abs(v).max(-1) / 127
        return np.divide(v, scale[:, None], where=scale[:, None] > 0, out=np.zeros_like(v)), scale
    # codes of 4 bits are at least 6: a group's scale is at most its smallest magnitude / 6
    g = np.abs(v.reshape(len(v), -1, 64))
    scale = (g.min(-1) / 6).max(-1)
    return np.full_like(v, 127.0) * (scale > 0)[:, None], scale


def check_tight(c, got, q, rows, scale=None, sums=0.0):
    """Outputs of tokens that see all of `rows` (keys, values), without room for anything absolute: the bound of kv_pool_ref.attend, and what weights
    lose as halves: the largest weight times scale of those that share a maximum is kept at 2^7 or more (2^6 for the logarithm's rounding and
    the like), and the smallest step of a half is 2^-24, so each weight times scale is off by at most 2^-25 / 2^6 of the largest.  bf16 calls over
    4-bit rows of two groups may round codes like the queries."""
    k, v = rows
    d, heads = c.d, q.shape[1]
    half = HALF[c.dtype] * (2 if (c.dtype, d, c.bits) == ("bf16", 128, 4) else 1)
    scale = d ** -0.5 if scale is None else scale
    for t in range(len(q)):
        for h in range(heads):
            kv = h * c.kh // heads
            want, bound = ref.attend(q[t, h:h + 1], k[:, kv:kv + 1], v[:, kv:kv + 1], scale, half)
            s = k[:, kv].astype(np.float64) @ ref.rotate(q[t, h].astype(np.float64)) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            code, of = value_parts(v[:, kv].astype(np.float64), c.bits)
            lost = 2.0 ** -31 * (p * np.maximum(of, 2.0 ** -64)).max() * np.linalg.norm(np.abs(code).sum(0).reshape(-1, 64), axis=-1) + sums * np.linalg.norm((p @ np.abs(v[:, kv])).reshape(-1, 64), axis=-1)
            off = np.linalg.norm((got[t, h] - want[0]).reshape(-1, 64), axis=-1)
            allowed = (bound[0] + lost) * (1 + OUT[c.dtype]) + OUT[c.dtype] * np.linalg.norm(want[0].reshape(-1, 64), axis=-1)
            if c.dtype == "f16":
                allowed += 8 * 2.0 ** -25
            assert (off <= allowed).all(), (t, h, off, allowed)


def rewrite(c, k, v, prefix):
    """The rows of the prefix, or of sequence 0, become k and v; what is stored of them."""
    pages, n = (c.prefix_pages if prefix else c.table[0]), len(k)
    at = np.arange(n)
    c.store(pages[at // c.page].astype(np.int64) * c.page + at % c.page, k, v)
    return ref.stored(k, c.bits).reshape(k.shape), ref.stored(v, c.bits).reshape(v.shape)


PLACES = [("own", 1, 2011), ("own", 3, 8000), ("prefix", 3, 700), ("prefix", 64, 8200), ("prefix", 200, 8200), ("prefix", 300, 2560)]


def place(ctx, where, tokens, n, d, bits, dtype, kh=1):  # noqa: F811
    """Rows of `n` positions that `tokens` tokens see: of a sequence, of a prefix for few rows, or of one for many (rows of one tile, of two and more)."""
    far = where == "prefix"
    c = Cache(ctx, [0 if far else n], kh, d, bits, 64, dtype, prefix=n if far else 0)
    return c, lambda q, **over: c.attend(q, [0 if far else n] * tokens, [0] * tokens, **over)


@pytest.mark.parametrize("d,bits", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("where,tokens,n", PLACES)
def test_values_of_zero_with_most_of_the_weight(ctx, d, bits, dtype, where, tokens, n):  # noqa: F811
    """Every 41st row has values of zero and a score far above the others (a null token): all of the output comes from the others."""
    c, attend = place(ctx, where, tokens, n, d, bits, dtype)
    rng = c.rng
    one = rng.standard_normal(d)
    q = rounded((one + 0.01 * rng.standard_normal((tokens, 1, d))), dtype)
    for above, size in ((0, 1e-4), (14, 1e-2), (18, 1.0), (24, 1e-4)):
        k, v = rng.standard_normal((n, 1, d)) * 0.02, rng.standard_normal((n, 1, d)) * size
        k[::41] = one * above * np.log(2) * d ** 0.5 / (one @ one)
        v[::41] = 0
        rows = rewrite(c, rounded(k, dtype), rounded(v, dtype), where == "prefix")
        assert not rows[1][::41].any() and rows[1][1].any()
        pick = rng.permutation(tokens)[:3]
        check_tight(c, attend(q)[pick], q[pick], rows)
    rows = rewrite(c, rounded(k, dtype), np.zeros_like(rounded(v, dtype)), where == "prefix")          # nothing else
    assert not attend(q).any()


@pytest.mark.parametrize("where,kh,tokens,n", [("own", 1, 600, 8000), ("prefix", 1, 3, 8000), ("prefix", 4, 2400, 8200)])
def test_weights_of_fp32_calls_keep_their_digits(ctx, where, kh, tokens, n):  # noqa: F811
    """The first 64 values of a few rows, the last 64 of all others, whose scale is far below: as halves on a grid of 2^-24 of the largest their
    weights would all be off by the same part.  Beside the bound: a sum of equal terms in fp32 is off by a step of 2^-23 an addition, of
    which an accumulator has fewer than one in 16 rows."""
    c, attend = place(ctx, where, tokens, n, 128, 8, "f32", kh)
    one = c.rng.standard_normal((1, kh, 128)).astype(np.float32)
    v = np.repeat(np.float32(48.5 * 2.0 ** -24) * one, n, 0)
    v[:, :, :64] = 0
    v[::2003, :, :64], v[::2003, :, 64:] = one[:, :, :64], 0
    rows = rewrite(c, np.zeros_like(v), v, where == "prefix")
    q = c.queries(tokens, kh)
    pick = c.rng.permutation(tokens)[:3]
    check_tight(c, attend(q)[pick], q[pick], rows, sums=n / 16 * 2.0 ** -23)


# ------------------------------------------------------------------------------------------------ pages outside the pool
@pytest.mark.parametrize("d,bits", SHAPES)
def test_choice_leaves_pages_outside_the_pool_to_the_last(ctx, d, bits):  # noqa: F811
    """Their positions are out of sight, so any other page comes before them, also one that scores below zero."""
    from kronos_2t_b200 import KronosCudaError
    page, n = 16, 12 * 16
    c = Cache(ctx, [n], 1, d, bits, page, "f32", block_keys=True)
    k = np.repeat(c.rng.standard_normal((1, 1, d)), n, 0) * np.repeat(1 + np.arange(12) / 8, page)[:, None, None]
    k = k.astype(np.float32)
    rewrite(c, k, k, False)
    q = -k[:1].reshape(1, 1, d)                     # the first page scores best
    assert c.select(q, [n], 6, 0, 1)[0, 0].tolist() == [0, 1, 2, 3, 4, 11]
    for bad in (-1, c.pool.num_pages, 1 << 30):
        c.table[0, [1, 7]] = bad
        got = [c.select(q, [n], top, 0, 1)[0, 0].tolist() for top in (6, 10, 11)]
        with pytest.raises(KronosCudaError, match="outside the pool"):
            ctx.synchronize()
        assert got == [[0, 2, 3, 4, 5, 11], [0, 2, 3, 4, 5, 6, 8, 9, 10, 11], [0, 1, 2, 3, 4, 5, 6, 8, 9, 10, 11]]
    ctx.synchronize()


def test_calls_without_a_token(ctx):  # noqa: F811
    c = Cache(ctx, [20], 2, 64, 8, 16, "bf16", block_keys=True)
    launches = ctx.launch_count
    c.pool.store_dev("bf16", 0, 0, 0, 0)
    c.pool.load_dev("f32", 0, 0, 0, 0)
    c.pool.attend_dev("bf16", 4, 0, 0, 0, 0, 3, 0, (0, 0), d_prefix_pages=0, prefix_len=50)
    c.pool.select_dev("bf16", 4, 0, 0, 0, 0, 3, 5, 0)
    c.pool.attend_chosen_dev("bf16", 4, 0, 0, 0, 0, 3, 5, 0, 0, (0, 0))
    ctx.synchronize()
    assert ctx.launch_count == launches


# ------------------------------------------------------------------------------------------------ the prefix of many rows
MANY = [(64, 8200), (200, 3000)]                    # rows of one tile and of two, both for the kernel of many rows


@pytest.mark.parametrize("d,bits", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tokens,n", MANY)
def test_a_row_of_a_prefix_that_is_not_finite(ctx, d, bits, dtype, tokens, n):  # noqa: F811
    """A key reaches every query of its kv head, a value likewise; a query that is not finite reaches its own row alone."""
    c = Cache(ctx, [3] * 2, 2, d, bits, 64, dtype, prefix=n)
    q = c.queries(tokens, 2)
    lens, seq = [3] * tokens, np.arange(tokens) % 2
    hurt = q.copy()
    hurt[5, 1, 3] = np.inf
    hurt[7, 0, d - 1] = np.nan
    got = c.attend(hurt, lens, seq)
    assert np.isnan(got[5, 1]).all() and np.isnan(got[7, 0]).all()
    keep = np.ones((tokens, 2), bool)
    keep[5, 1] = keep[7, 0] = False
    assert np.isfinite(got[keep]).all()
    c.check(got[:4], q[:4], lens[:4], seq[:4])
    good, bad = np.ones((1, 2, d), np.float32), np.ones((1, 2, d), np.float32)
    bad[0, 1, 9] = np.nan
    for at, (k, v) in ((n - 1, (bad, good)), (70, (good, bad))):
        slot = np.array([int(c.prefix_pages[at // 64]) * 64 + at % 64])
        c.store(slot, k, v)
        got = c.attend(q, lens, seq)
        assert np.isnan(got[:, 1]).all() and np.isfinite(got[:, 0]).all()
        c.store(slot, good, good)
        assert np.isfinite(c.attend(q, lens, seq)).all()


@pytest.mark.parametrize("d,bits", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("where,tokens,n", [("own", 3, 700), ("prefix", 64, 8200), ("prefix", 200, 3000)])
def test_scales_far_apart_and_queries_of_all_sizes(ctx, d, bits, dtype, where, tokens, n):  # noqa: F811
    c, attend = place(ctx, where, tokens, n, d, bits, dtype)
    rng = c.rng
    k, v = (rng.standard_normal((n, 1, d)) for _ in range(2))
    v *= 10.0 ** rng.integers(-6, 7, (n, 1, 1))
    v[::7], k[::11] = 0, 0
    rows = rewrite(c, rounded(k, dtype), rounded(v, dtype), where == "prefix")
    q = rng.standard_normal((tokens, 2, d)) * 1.5
    pick = rng.permutation(tokens)[:2]
    for size in (0.0, 1e-30, 1e-3, 1.0, 3.0):
        x = rounded(q * size, dtype)
        check_tight(c, attend(x)[pick], x[pick], rows)
    x = rounded(q, dtype)
    check_tight(c, attend(x, scale=0.31)[pick], x[pick], rows, scale=0.31)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tokens,n", [(3, 200)] + MANY)
def test_strided_rows_behind_a_prefix(ctx, dtype, tokens, n):  # noqa: F811
    """Heads outermost, at addresses that allow no wide access; what lies between the rows stays as it was."""
    import torch
    d, heads = 64, 4
    c = Cache(ctx, [5] * tokens, 2, d, 8, 16, dtype, prefix=n)
    q, lens = c.queries(tokens, heads), [5] * tokens
    straight = c.attend(q, lens)
    wide = torch.full((heads, tokens, d + 3), 2.0, device="cuda", dtype=torch_type(dtype))
    wide[:, :, 1:d + 1] = device(q, dtype).transpose(0, 1)
    out, dl, dt, far = torch.full_like(wide, 9.0), device(np.array(lens, np.int32)), device(c.table), device(c.prefix_pages)
    work, size = torch.empty(c.pool.workspace_bytes(heads, tokens, n), dtype=torch.uint8, device="cuda"), wide.element_size()
    c.pool.attend_dev(dtype, heads, tokens, (wide.data_ptr() + size, d + 3, tokens * (d + 3)), dl.data_ptr(), dt.data_ptr(), dt.shape[1],
                      (out.data_ptr() + size, d + 3, tokens * (d + 3)), (work.data_ptr(), work.numel()), d_prefix_pages=far.data_ptr(), prefix_len=n)
    ctx.synchronize()
    got = out.float().cpu().numpy()
    assert np.array_equal(got[:, :, 1:d + 1].transpose(1, 0, 2), straight)
    assert (got[:, :, 0] == 9).all() and (got[:, :, d + 1:] == 9).all()


# ------------------------------------------------------------------------------------------------ other calls
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bits", [8, 4])
def test_strided_rows_of_other_types(ctx, dtype, bits):  # noqa: F811
    """Rows in and out, and queries of a choice, at odd places of a wider buffer."""
    import torch
    d, kh, heads, n, page = 128, 2, 6, 75, 16
    c = Cache(ctx, [n], kh, d, bits, page, dtype, block_keys=True)
    k, v = (rounded(c.rng.standard_normal((n, kh, d)), dtype) for _ in range(2))
    wide = [torch.full((n, kh, d + 5), 2.0, device="cuda", dtype=torch_type(dtype)) for _ in range(4)]
    wide[0][:, :, 3:d + 3], wide[1][:, :, 3:d + 3] = device(k, dtype), device(v, dtype)
    rows = [(w.data_ptr() + 3 * w.element_size(), kh * (d + 5), d + 5) for w in wide]
    at = np.arange(n)
    slots = device(c.table[0][at // page].astype(np.int64) * page + at % page)
    c.pool.store_dev(dtype, rows[0], rows[1], slots.data_ptr(), n)
    c.pool.load_dev(dtype, slots.data_ptr(), n, rows[2], rows[3])
    ctx.synchronize()
    for x, w in ((k, wide[2]), (v, wide[3])):
        got = w.float().cpu().numpy()
        assert np.array_equal(got[:, :, 3:d + 3], rounded(ref.read_back(x, bits).reshape(n, kh, d), dtype))
        assert (got[:, :, :3] == 2).all() and (got[:, :, d + 3:] == 2).all()
    q, lens = c.queries(4, heads), [n, 40, 3, n - 1]
    want = c.select(q, lens, 3, 0, 1, seq=[0] * 4)
    x = torch.full((heads, 4, d + 7), 2.0, device="cuda", dtype=torch_type(dtype))
    x[:, :, 1:d + 1] = device(q, dtype).transpose(0, 1)
    dl, dt, ds, out = device(np.array(lens, np.int32)), device(c.table), device(np.zeros(4, np.int32)), torch.full((4, kh, 3), 77, dtype=torch.int32, device="cuda")
    c.pool.select_dev(dtype, heads, 4, (x.data_ptr() + x.element_size(), d + 7, 4 * (d + 7)), dl.data_ptr(), dt.data_ptr(), dt.shape[1], 3, out.data_ptr(), sinks=0, local=1, d_seq=ds.data_ptr())
    ctx.synchronize()
    assert np.array_equal(out.cpu().numpy(), want)


@pytest.mark.parametrize("dtype,d,bits", [("bf16", 128, 8), ("f32", 64, 4)])
def test_a_page_named_twice_counts_twice(ctx, dtype, d, bits):  # noqa: F811
    page, n = 16, 70
    c = Cache(ctx, [n], 2, d, bits, page, dtype)
    q = c.queries(1, 4)
    chosen = np.array([[[1, 3, 1, -1, 4], [4, 4, 0, 0, 0]]], np.int32)
    rows = [np.concatenate([np.arange(p * page, min(n, (p + 1) * page)) for p in x if p >= 0]) for x in chosen[0]]
    c.check(c.attend(q, [n], chosen=chosen), q, [n], rows_of=lambda t, h: rows[h])


@pytest.mark.parametrize("kh,heads,d,bits,prefix", [(256, 256, 64, 8, 0), (256, 256, 64, 4, 40), (1, 256, 64, 4, 0), (1, 256, 64, 4, 3000), (2, 512, 128, 8, 40), (2, 512, 128, 8, 3000)])
def test_most_heads(ctx, kh, heads, d, bits, prefix):  # noqa: F811
    """256 kv heads, and 256 query heads of one."""
    c = Cache(ctx, [20, 0, 37], kh, d, bits, 16, "bf16", prefix=prefix, block_keys=True)
    q = c.queries(3, heads)
    lens = [20, 0, 37]
    got = c.attend(q, lens)
    some = [0, 1, kh // 2, kh - 1]
    for h in set(some):
        mine = slice(h * heads // kh, (h + 1) * heads // kh)
        for t in range(3):
            k, v = (np.concatenate((c.far[i][:, h:h + 1], c.own[t][i][:, h:h + 1])) for i in range(2))
            want, bound = ref.attend(q[t, mine], k, v, d ** -0.5, HALF["bf16"])
            off = np.linalg.norm((got[t, mine] - want).reshape(-1, d // 64, 64), axis=-1)
            assert (off <= bound * (1 + OUT["bf16"]) + OUT["bf16"] * np.linalg.norm(want.reshape(-1, d // 64, 64), axis=-1) + 1e-7).all()
    pages = c.select(q, lens, 2, 0, 1)
    assert (pages[0] == [0, 1]).all() and (pages[1] == -1).all() and (pages[2, :, 1] == 2).all()


@pytest.mark.parametrize("d,bits", SHAPES)
@pytest.mark.parametrize("n,kh", [(9001, 4), (1301, 5), (20003, 2)])
def test_many_rows(ctx, d, bits, n, kh):  # noqa: F811
    """As many as one and two rows on their way a thread are for, the last CTA's part full; every fifth token is left out."""
    import torch

    from kronos_2t_b200 import KvPool
    rng = np.random.default_rng(n)
    pages = -(-n // 64) + 2
    slots = rng.permutation(pages * 64)[:n].astype(np.int64)
    slots[::5] = -1
    x = [rounded(rng.standard_normal((n, kh, d)), "bf16") for _ in range(2)]
    pool, dx, ds = KvPool(ctx, kh, d, bits, 64, pages), [device(a, "bf16") for a in x], device(slots)
    pool.store_dev("bf16", dx[0].data_ptr(), dx[1].data_ptr(), ds.data_ptr(), n)
    out = [torch.full((n, kh, d), 5.0, device="cuda") for _ in x]
    pool.load_dev("f32", ds.data_ptr(), n, out[0].data_ptr(), out[1].data_ptr())
    ctx.synchronize()
    for a, o in zip(x, out):
        want = ref.read_back(a, bits).reshape(n, kh, d)
        want[::5] = 5.0
        assert np.array_equal(o.cpu().numpy(), want)
