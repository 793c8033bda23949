"""The shared pool of cached keys and values on the device, at the ends of what its calls allow."""
import os
import subprocess
import sys

import numpy as np
import pytest

import kv_pool_ref as ref
from test_gpu_kv_pool import HALF, OUT, SHAPES, Cache, ctx, rounded  # noqa: F401

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
