"""The shared pool of cached keys and values without a device: struct layouts, refusals, and the restatement against the oracle."""
import ctypes as C

import numpy as np
import pytest

import kv_pool_ref as ref
from k2t_internal import internal
from test_boundary_structs import ctypes_struct, header_struct, rust_struct, same


@pytest.mark.parametrize("name,cls", [("KronosCudaKvPoolConfig", "KvPoolConfig"), ("KronosCudaRows", "Rows"), ("KronosCudaPoolAttention", "PoolAttention")])
def test_struct_layouts_agree(name, cls):
    from kronos_2t_b200 import ffi
    h, r, c = header_struct(name), rust_struct(name), ctypes_struct(getattr(ffi, cls))
    assert len(h) >= 3 and h == r and same(h, c)


def config(**over):
    from kronos_2t_b200 import ffi
    c = dict(struct_size=C.sizeof(ffi.KvPoolConfig), kv_heads=4, head_dim=128, kv_bits=8, page_tokens=64, num_pages=10, flags=1)
    c.update(over)
    return ffi.KvPoolConfig(**c)


def arguments(**over):
    from kronos_2t_b200 import ffi
    rows = ffi.Rows(1 << 20, 0, 0)
    a = dict(struct_size=C.sizeof(ffi.PoolAttention), row_type=1, heads=28, n_tok=3, pages_stride=5, q=rows, out=rows, lens=4096, pages=4096, workspace=1 << 20, workspace_bytes=1 << 40)
    a.update(over)
    return ffi.PoolAttention(**a)


def refusal(cfg, args=None, what=0):
    f = internal("pool_refusal", C.c_char_p, C.c_void_p, C.c_void_p, C.c_int32)
    got = f(C.byref(cfg), None if args is None else C.byref(args), what)
    return None if got is None else got.decode()


@pytest.mark.parametrize("over,message", [
    (dict(struct_size=4), "struct_size"), (dict(kv_heads=0), "kv heads"), (dict(kv_heads=257), "kv heads"), (dict(head_dim=96), "head_dim"), (dict(head_dim=256), "head_dim"),
    (dict(kv_bits=5), "kv_bits"), (dict(page_tokens=8), "page_tokens"), (dict(page_tokens=48), "page_tokens"), (dict(page_tokens=256), "page_tokens"),
    (dict(num_pages=0), "pages"), (dict(num_pages=1 << 31), "pages"), (dict(flags=2), "flag")])
def test_configurations_that_are_refused(over, message):
    assert refusal(config()) is None
    assert message in refusal(config(**over))


def rows(data, token=0, head=0):
    from kronos_2t_b200 import ffi
    return ffi.Rows(data, token, head)


@pytest.mark.parametrize("over,message", [
    (dict(struct_size=4), "struct_size"), (dict(heads=30), "heads"), (dict(heads=0), "heads"), (dict(heads=4 * 257), "heads"), (dict(n_tok=(1 << 20) + 1), "tokens"),
    (dict(lens=None), "NULL"), (dict(pages=None), "NULL"), (dict(pages_stride=0), "pages_stride"), (dict(prefix_len=5), "without its pages"), (dict(prefix_len=1 << 31, prefix_pages=4096), "prefix"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(row_type=3), "type"), (dict(q=rows(None)), "q is NULL"), (dict(out=rows(None)), "out is NULL"),
    (dict(q=rows((1 << 20) + 1)), "aligned"), (dict(out=rows(1 << 20, 128, 128)), "overlap"), (dict(out=rows(1 << 20, 28 * 128, 64)), "overlap"), (dict(q=rows(1 << 20, 1 << 40)), "stride"),
    (dict(workspace=None), "workspace"), (dict(workspace=(1 << 20) + 8), "workspace"), (dict(workspace_bytes=64), "workspace"), (dict(top=4), "attend takes no chosen"), (dict(chosen=4096), "attend takes no chosen")])
def test_attention_calls_that_are_refused(over, message):
    assert refusal(config(), arguments()) is None
    assert refusal(config(), arguments(out=rows(1 << 20, 128, 3 * 128))) is None          # heads outermost
    assert message in refusal(config(), arguments(**over))


@pytest.mark.parametrize("what,over,message", [
    (1, dict(chosen=None), "chosen is NULL"), (1, dict(top=0), "top"), (1, dict(top=32769), "top"), (1, dict(prefix_len=3, prefix_pages=4096), "prefix"), (2, dict(local=0), "local"),
    (2, dict(sinks=4), "sinks"), (2, dict(sinks=0xffffffff), "sinks"), (2, dict(local=0xffffffff), "local"), (2, dict(pages_stride=32769), "32768")])
def test_choices_that_are_refused(what, over, message):
    good = dict(chosen=4096, top=4, sinks=1, local=1)
    assert refusal(config(), arguments(**good), what) is None
    assert message in refusal(config(), arguments(**{**good, **over}), what)


def test_choice_needs_block_keys():
    assert "block keys" in refusal(config(flags=0), arguments(chosen=4096, top=4, sinks=1, local=1), 2)


def test_calls_without_a_token_need_nothing():
    assert refusal(config(), arguments(n_tok=0, workspace=None, workspace_bytes=0)) is None
    assert refusal(config(), arguments(n_tok=0, workspace=None, workspace_bytes=0, prefix_len=1000, prefix_pages=4096)) is None
    assert refusal(config(), arguments(n_tok=0, workspace=None, workspace_bytes=0, chosen=4096, top=3), 1) is None
    assert "prefix too long" in refusal(config(), arguments(n_tok=1 << 20, prefix_len=(1 << 31) - 1, prefix_pages=4096))


def test_calls_without_a_token_take_empty_buffers():
    """An empty tensor has no address."""
    none = dict(n_tok=0, q=rows(None), out=rows(None), lens=None, pages=None, workspace=None, workspace_bytes=0)
    assert refusal(config(), arguments(**none)) is None
    assert refusal(config(), arguments(**none, prefix_len=1000)) is None
    for what in (1, 2):
        assert refusal(config(), arguments(**none, top=3, sinks=1, local=1), what) is None
    assert "type" in refusal(config(), arguments(**none, row_type=3))
    assert "heads" in refusal(config(), arguments(**{**none, "heads": 30}))


@pytest.mark.parametrize("kv_heads,head_dim,bits,heads", [(4, 128, 8, 28), (1, 64, 4, 20), (8, 128, 4, 64), (3, 64, 8, 3)])
def test_workspaces_cover_what_calls_need(kv_heads, head_dim, bits, heads):
    """A call is refused one byte below the size that is asked for some type, never at it; with a prefix it is enough without one."""
    f = internal("pool_work_bytes", C.c_size_t, C.c_void_p, C.c_uint32, C.c_uint32, C.c_uint32, C.c_uint32)
    shape = (C.c_uint32 * 6)(kv_heads, head_dim, bits, 6, 10, 1)
    cfg = config(kv_heads=kv_heads, head_dim=head_dim, kv_bits=bits)
    for n_tok in (1, 2, 3, 7, 40, 160, 2000):
        for prefix in (0, 1, 500, 100000):
            need = f(shape, heads, n_tok, prefix, 148)
            assert need >= f(shape, heads, n_tok, 0, 148) > 0
            for stride in (1, 3, 40, 5000):
                for row_type in (0, 1, 2):
                    a = dict(heads=heads, n_tok=n_tok, prefix_len=prefix, prefix_pages=4096, pages_stride=stride, row_type=row_type)
                    assert refusal(cfg, arguments(**a, workspace_bytes=need)) is None
                    assert "workspace too small" in refusal(cfg, arguments(**a, workspace_bytes=need - 1))


@pytest.mark.parametrize("heads,n_tok,prefix,refused", [
    (28, 3, 1000, False), (30, 3, 0, True), (0, 3, 0, True), (4 * 257, 3, 0, True), (28, 1 << 20, 0, False), (28, (1 << 20) + 1, 0, True), (1024, 1 << 20, 0, False),
    (28, 3, (1 << 31) - 1, False), (28, 3, 1 << 31, True), (28, 3, (1 << 32) - 1, True), (1024, 1 << 20, 16383, True), (28, 1 << 20, 600000, True)])
def test_workspaces_of_sizes_that_are_refused(heads, n_tok, prefix, refused):
    """0, as the header says: what attention refuses is not planned."""
    f = internal("pool_workspace", C.c_size_t, C.c_void_p, C.c_uint32, C.c_uint32, C.c_uint32, C.c_uint32)
    shape = (C.c_uint32 * 6)(4, 128, 8, 6, 10, 1)
    size = f(shape, heads, n_tok, prefix, 148)
    assert (size == 0) == refused
    call = refusal(config(), arguments(heads=heads, n_tok=n_tok, prefix_len=prefix, prefix_pages=4096, workspace_bytes=size))
    assert (call is not None) == refused


def test_lines_of_tiles_are_counted_in_32_bits():
    """The tiles of all items, with a CTA's part of them behind, stay below 2^32: the limit is as far below it as the largest part is long."""
    most = dict(n_tok=1 << 20, heads=1024, prefix_pages=4096, workspace_bytes=1 << 63)
    assert refusal(config(), arguments(**most, prefix_len=64 * 251 - 1)) is None
    assert "so many tokens" in refusal(config(), arguments(**most, prefix_len=64 * 251))
    few = dict(n_tok=1, heads=256, prefix_pages=4096, workspace_bytes=1 << 63)          # 256 kv heads: (4 + 256) tiles a 64 positions
    last = 64 * ((1 << 32) - (1 << 26)) // 260 // 64 * 64
    assert refusal(config(kv_heads=256), arguments(**few, prefix_len=last - 64)) is None
    assert "so many tokens" in refusal(config(kv_heads=256), arguments(**few, prefix_len=last))
    assert (1 << 32) - (1 << 26) + ((1 << 32) - (1 << 26)) // 64 < 1 << 32


def test_null_handles_are_tolerated():
    import kronos_2t_b200 as k2
    L = k2.load_library()
    assert L.kronos_cuda_kv_pool_create(None, None) is None
    L.kronos_cuda_kv_pool_free(None, None)
    assert L.kronos_cuda_kv_pool_bytes(None) == 0 and L.kronos_cuda_kv_pool_workspace(None, 4, 1, 0) == 0
    assert L.kronos_cuda_kv_pool_store_dev(None, None, 0, None, None, None, 1) == -1
    assert L.kronos_cuda_kv_pool_load_dev(None, None, 0, None, None, None, 1) == -1
    for f in (L.kronos_cuda_kv_pool_attend_dev, L.kronos_cuda_kv_pool_attend_chosen_dev, L.kronos_cuda_kv_pool_select_dev):
        assert f(None, None, None) == -1


def test_restatement_against_the_oracle(oracle):
    """Transform and 4-bit assignment are the oracle's; the inverse undoes the transform; quantised rows are near what they stand for."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((7, 128)).astype(np.float32)
    want = np.stack([oracle.fwht64(row, 0) for row in x])
    assert np.array_equal(ref.rotate(x), want)
    assert np.abs(ref.rotate_back(ref.rotate(x.astype(np.float64))) - x).max() < 1e-12
    # 8 bits: half a step of max / 127 per transformed value, so its 2-norm over 64 values at most 4 steps of the largest
    assert np.abs(ref.stored(x, 8) - want).max() <= np.abs(want).max() / 127 * 0.5001
    # 4 bits: centroids are at most 16 half steps of 1/127 apart from their borders, plus the fitted scale
    assert np.abs(ref.stored(x, 4) - want).max() <= np.abs(want).max() * 0.25


@pytest.mark.parametrize("d", [64, 128])
def test_codes_and_scales_are_the_oracles(oracle, d):
    """Bit for bit, of both widths of codes: ordinary rows of many sizes, rows of zeros and below what is kept, values that are codes."""
    rng = np.random.default_rng(d)
    x = (rng.standard_normal((400, d)) * 10.0 ** rng.uniform(-8, 8, (400, 1))).astype(np.float32)
    x[::50] = 0
    x[1::50] = np.float32(1e-9)
    x[2::50] = ref.rotate_back(np.tile(ref.CENTROIDS * np.float32(0.5), d // 16)[None]).astype(np.float32)
    x[3::50] = rng.integers(-3, 4, d)
    code8, scale8 = ref.quant8(ref.rotate(x))
    code4, scale4 = ref.quant4(ref.rotate(x))
    for i, row in enumerate(x):
        q, s = oracle.kv_quant_head(row)
        assert np.array_equal(q, code8[i]) and s == scale8[i], i
        q, s = oracle.kv_quant_head_q4(row)
        nibbles = np.stack((q.reshape(-1, 16) & 15, q.reshape(-1, 16) >> 4), 1).reshape(-1)          # 16 low ones, then 16 high ones
        assert np.array_equal(ref.CENTROIDS[nibbles], code4[i]), i
        assert np.array_equal((s.astype(np.uint32) << 16).view(np.float32), scale4[i]), i
