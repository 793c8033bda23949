"""The operators on a pool of cached keys and values that many sequences share (kronos_2t_b200.ffi.KvPool), as cases that can be timed
and compared.  `run` computes them in elementary torch operations, or, with `own`, by the framework's calls.

Kinds
  cache    rows of keys and values are quantised into their slots and read back
  prefix   attention of `seqs` sequences (`new` query tokens each) over one prefix that all of them see and over their own rows
  sparse   attention of a token over the `top` pages of its sequence that score best against block keys, the first and last ones among them

Rows are kept in the format of the engines' caches.  Per 64 values: signs of a hash, Walsh-Hadamard transform over eight.  8 bits: one
fp32 scale per row.  4 bits: 16 centroids, one bf16 scale per 64 values by least squares over a first assignment.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token of the smallest shape goes into the cache: launches and latency
        dict(name="cache_step", kind="cache", n_tok=1, kv_heads=3, head_dim=64, bits=8, page=16, dtype="f32", spread=True, block_keys=False),
        # a decode batch, one token of each sequence, each in a page of its own
        dict(name="cache_batch", kind="cache", n_tok=96, kv_heads=4, head_dim=128, bits=4, page=64, dtype="bf16", spread=True, block_keys=False),
        # a long prompt is written, with the block keys of its pages
        dict(name="cache_prompt", kind="cache", n_tok=16384, kv_heads=8, head_dim=128, bits=8, page=64, dtype="bf16", spread=False, block_keys=True),
        # a prompt of odd length, as many key heads as query heads, 4 bits
        dict(name="cache_prompt_q4", kind="cache", n_tok=4001, kv_heads=32, head_dim=64, bits=4, page=32, dtype="f16", spread=False, block_keys=False),
        # three short answers behind a short instruction, small model, fp32 rows as the projections leave them
        dict(name="prefix_short", kind="prefix", seqs=3, new=1, prefix=150, own=40, heads=9, kv_heads=3, head_dim=64, bits=8, page=16, dtype="f32"),
        # a chat server's decode step behind a system prompt
        dict(name="prefix_chat", kind="prefix", seqs=24, new=1, prefix=2000, own=700, heads=28, kv_heads=4, head_dim=128, bits=8, page=64, dtype="bf16"),
        # many questions about one long document
        dict(name="prefix_many", kind="prefix", seqs=160, new=1, prefix=32768, own=1000, heads=64, kv_heads=8, head_dim=128, bits=8, page=64, dtype="bf16"),
        # few questions about a very long one, 4 bits
        dict(name="prefix_long_q4", kind="prefix", seqs=8, new=1, prefix=120000, own=500, heads=32, kv_heads=4, head_dim=128, bits=4, page=64, dtype="bf16"),
        # five drafted tokens of each sequence to verify at once
        dict(name="prefix_verify", kind="prefix", seqs=16, new=5, prefix=6001, own=300, heads=32, kv_heads=4, head_dim=128, bits=8, page=32, dtype="f16"),
        # one sequence behind a long context, a decode step
        dict(name="sparse_step", kind="sparse", seqs=1, new=1, ctx=30000, top=16, sinks=1, local=2, heads=28, kv_heads=4, head_dim=128, bits=8, page=64, dtype="bf16"),
        # a decode step of a ragged batch
        dict(name="sparse_batch", kind="sparse", seqs=48, new=1, ctx=40000, top=32, sinks=1, local=4, heads=32, kv_heads=4, head_dim=128, bits=8, page=64, dtype="f16"),
        # the tokens of a prompt, each with its own choice
        dict(name="sparse_prompt", kind="sparse", seqs=1, new=2000, ctx=8000, top=24, sinks=1, local=2, heads=32, kv_heads=4, head_dim=128, bits=4, page=32, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "prefix", "prefix", "sparse", "sparse"])
    head_dim, kv_heads, group = rng.choice([64, 128, 128]), rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([1, 2, 3, 4, 6, 7, 8, 16])
    shape = dict(kind=kind, kv_heads=kv_heads, head_dim=head_dim, bits=rng.choice([8, 8, 4]), page=rng.choice([16, 32, 64, 64, 128]),
                 dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    if kind == "cache":
        return dict(shape, n_tok=_log(rng, 1, 16000), spread=rng.random() < 0.4, block_keys=rng.random() < 0.5)
    shape["heads"] = kv_heads * group
    if kind == "prefix":
        new, prefix = rng.choice([1, 1, 1, 2, 3, 8]), _log(rng, 1, 100000)
        seqs = _log(rng, 1, max(1, min(160, int(3e8 / (new * shape["heads"] * prefix)))))
        return dict(shape, seqs=seqs, new=new, prefix=prefix, own=_log(rng, new, 1000))
    new = rng.choice([1, 1, 1, _log(rng, 2, 1200)])
    seqs = 1 if new > 1 else _log(rng, 1, 48)
    top = rng.randint(4, 32)
    return dict(shape, seqs=seqs, new=new, ctx=max(new, _log(rng, 100, min(40000, 2000000 // (seqs * kv_heads)))), top=top, sinks=rng.randint(0, 2), local=rng.randint(1, 2))


# ------------------------------------------------------------------------------------------------ inputs
def _pages(n, page):
    return (n + page - 1) // page


def _inputs(case, seed):
    """Keys, values and queries of the case and where their rows go: for kind `cache` the slots of the tokens; else a table of pages
    per sequence (-1 behind its last), the rows that a token sees of its own sequence, and the pages of the prefix."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    page, kh, d, dtype = case["page"], case["kv_heads"], case["head_dim"], TYPES[case["dtype"]]

    def rows(n, heads, spread):
        x = torch.randn(n, heads, d, generator=gen, device="cuda")
        if spread:          # some channels of keys are large throughout
            x = x * (1.0 + 4.0 * (torch.rand(heads, d, generator=gen, device="cuda") > 0.95))
        return x

    if case["kind"] == "cache":
        n = case["n_tok"]
        num = n + 3 if case["spread"] else _pages(n, page) + 3
        order = torch.randperm(num, generator=cpu)
        if case["spread"]:
            slots = order[:n] * page + torch.randint(page, (n,), generator=cpu)
        else:
            at = torch.arange(n)
            slots = order[at // page] * page + at % page
        return dict(k=rows(n, kh, True).to(dtype), v=rows(n, kh, False).to(dtype), slots=slots.cuda(), num_pages=num)
    seqs, new, heads = case["seqs"], case["new"], case["heads"]
    longest, prefix = (case["own"], case["prefix"]) if case["kind"] == "prefix" else (case["ctx"], 0)
    shortest = new if case["kind"] == "prefix" else max(new, longest // 10)
    lens = torch.randint(shortest, longest + 1, (seqs,), generator=cpu)
    lens[0] = longest
    counts = [_pages(int(n), page) for n in lens]
    num = _pages(prefix, page) + sum(counts) + 2
    order = torch.randperm(num, generator=cpu)
    prefix_pages, at = order[:_pages(prefix, page)], _pages(prefix, page)
    table = torch.full((seqs, max(counts)), -1, dtype=torch.int32)
    slots = [(prefix_pages[torch.arange(prefix) // page] * page + torch.arange(prefix) % page)]
    for b, c in enumerate(counts):
        mine = order[at:at + c]
        at += c
        table[b, :c] = mine.int()
        j = torch.arange(int(lens[b]))
        slots.append(mine[j // page] * page + j % page)
    slots = torch.cat(slots).cuda()
    n = slots.numel()
    k, v = rows(n, kh, True), rows(n, kh, False)
    if case["kind"] == "sparse":        # neighbouring keys are alike, so that pages differ from one another
        drift = torch.randn(n // 256 + 2, kh, d, generator=gen, device="cuda")
        at = torch.arange(n, device="cuda") // 256
        k += drift[at]
    q = torch.randn(seqs * new, heads, d, generator=gen, device="cuda") * 1.5
    seen = (lens[:, None] - new + 1 + torch.arange(new)[None, :]).reshape(-1)
    seq = torch.arange(seqs).repeat_interleave(new)
    return dict(k=k.to(dtype), v=v.to(dtype), q=q.to(dtype), slots=slots, num_pages=num, table=table.cuda(), lens=seen.int().cuda(), seq=seq.int().cuda(),
                prefix_pages=prefix_pages.int().cuda(), max_len=longest)


# ------------------------------------------------------------------------------------------------ plain forms
_SIGNS = {}
_CENTROIDS = [-127, -96, -75, -58, -44, -31, -18, -6, 6, 18, 31, 44, 58, 75, 96, 127]
_EDGES = [12.0, 24.5, 37.5, 51.0, 66.5, 85.5, 111.5]


def _signs(d):
    """+-1 for every value of a row: the low bit of a SplitMix64 step per position, one stream per 64 values."""
    if d not in _SIGNS:
        mask, g, out = (1 << 64) - 1, 0x9E3779B97F4A7C15, []
        for i in range(d):
            z = (g + (i // 64) * 0xBF58476D1CE4E5B9 + (i % 64 + 1) * g) & mask
            z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & mask
            z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & mask
            out.append(-1.0 if (z ^ (z >> 31)) & 1 else 1.0)
        _SIGNS[d] = torch.tensor(out, device="cuda")
    return _SIGNS[d]


def _butterflies(x):
    shape, h = x.shape, 1
    while h < 64:
        x = x.reshape(-1, 64 // (2 * h), 2, h)
        a, b = x[:, :, 0], x[:, :, 1]
        x = torch.stack((a + b, a - b), 2)
        h *= 2
    return x.reshape(shape)


def _rotate(x):
    return _butterflies(x.float() * _signs(x.shape[-1]) * 0.125)


def _rotate_back(r):
    return _butterflies(r) * 0.125 * _signs(r.shape[-1])


def _ratio(a, b):
    """a / b rounded once (a division by a number known on the host is a product with its reciprocal)."""
    return torch.div(torch.as_tensor(a, dtype=torch.float32, device="cuda"), torch.as_tensor(b, dtype=torch.float32, device="cuda"))


def _quant8(r):
    top = r.abs().amax(-1, keepdim=True)
    some = top > 1.1920929e-07
    inv = torch.where(some, _ratio(127.0, top), 0.0)
    return torch.round(r * inv), torch.where(some, _ratio(top, 127.0), 0.0)


def _nearest(y):
    a, p = y.abs(), torch.zeros_like(y, dtype=torch.uint8)
    for e in _EDGES:
        p += a >= e
    return torch.where(y >= 0, 8 + p, 7 - p)


def _quant4(r):
    table = torch.tensor(_CENTROIDS, dtype=torch.float32, device="cuda")
    r = r.reshape(*r.shape[:-1], -1, 64)
    top = r.abs().amax(-1, keepdim=True)
    some = top >= 1e-30
    c = table[_nearest(r * torch.where(some, _ratio(127.0, top), 0.0)).int()]
    num, rc = torch.zeros_like(top), r * c
    for i in range(64):
        num = num + rc[..., i:i + 1]
    den = (c * c).sum(-1, keepdim=True)
    s = torch.where(num > 0, num / den, _ratio(top, 127.0)).bfloat16().float()
    i = _nearest(r * torch.where(s > 1e-30, _ratio(1.0, s), 0.0))
    i, s = torch.where(some, i, 8), torch.where(some, s, 0.0)
    return table[i.int()].flatten(-2), s.squeeze(-1)


class _Plain:
    """The pool as tensors: code values (whole numbers up to 127) and scales by slot, block keys by page."""

    def __init__(self, case, num_pages):
        n, kh, d = num_pages * case["page"], case["kv_heads"], case["head_dim"]
        self.bits, self.page, self.groups = case["bits"], case["page"], 1 if case["bits"] == 8 else d // 64
        self.codes = [torch.zeros(n, kh, d, dtype=torch.int8, device="cuda") for _ in range(2)]
        self.scales = [torch.zeros(n, kh, self.groups, device="cuda") for _ in range(2)]

    def store(self, slots, k, v):
        for i, x in enumerate((k, v)):
            code, scale = (_quant8 if self.bits == 8 else _quant4)(_rotate(x))
            self.codes[i][slots] = code.to(torch.int8)
            self.scales[i][slots] = scale

    def rotated(self, which, slots):
        c, s = self.codes[which][slots].float(), self.scales[which][slots]
        return (c.reshape(*c.shape[:-1], self.groups, -1) * s[..., None]).flatten(-2)

    def store_block_keys(self, num_pages):
        at = torch.arange(num_pages, device="cuda") * self.page
        total = torch.zeros(num_pages, *self.codes[0].shape[1:], device="cuda")
        for i in range(self.page):
            total = total + self.rotated(0, at + i)
        self.block_codes, self.block_scales = _quant8(total * (1.0 / self.page))


def _softmax_sum(s, v):
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, 1.0, total)


def _plain_prefix(case, x, pool):
    kh, d, page, t = case["kv_heads"], case["head_dim"], case["page"], x["q"].shape[0]
    g = case["heads"] // kh
    q = _rotate(x["q"]).reshape(t, kh, g, d) * d ** -0.5
    at = torch.arange(case["prefix"], device="cuda")
    slots = x["prefix_pages"].long()[at // page] * page + at % page
    pk, pv = (pool.rotated(i, slots).transpose(0, 1) for i in range(2))                    # [kv head][position][d]
    far = torch.matmul(q.transpose(0, 1).reshape(kh, t * g, d), pk.transpose(1, 2))
    width = x["table"].shape[1] * page
    at = torch.arange(width, device="cuda")
    out, step = torch.empty(t, kh, g, d, device="cuda"), max(1, int(2.5e8 / (kh * width * d)))
    for t0 in range(0, t, step):
        part = slice(t0, min(t, t0 + step))
        n = part.stop - t0
        seen = at[None] < x["lens"][part, None]
        own_slots = torch.where(seen, x["table"].long()[x["seq"][part].long()][:, at // page] * page + at % page, 0)
        k, v = (pool.rotated(i, own_slots).transpose(1, 2) for i in range(2))              # [token][kv head][row][d]
        near = torch.matmul(q[part], k.transpose(2, 3)).masked_fill(~seen[:, None, None], -math.inf)
        s = torch.cat((far.reshape(kh, t, g, -1)[:, part].transpose(0, 1), near), -1)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p[..., :case["prefix"]].transpose(0, 1).reshape(kh, n * g, -1), pv).reshape(kh, n, g, d).transpose(0, 1)
        o = o + torch.matmul(p[..., case["prefix"]:], v)
        out[part] = o / torch.where(total == 0, 1.0, total)
    return _rotate_back(out).reshape(t, kh * g, d).to(x["q"].dtype)


def _plain_sparse(case, x, pool):
    kh, d, page, t, top = case["kv_heads"], case["head_dim"], case["page"], x["q"].shape[0], case["top"]
    g, dev = case["heads"] // kh, "cuda"
    heads = x["q"].float().reshape(t, kh, g, d)
    total = heads[:, :, 0]
    for i in range(1, g):
        total = total + heads[:, :, i]
    code, _ = _quant8(_rotate(total))
    pages = (x["lens"] + page - 1) // page                       # of each token
    width = x["table"].shape[1]
    at = torch.arange(width, device=dev)
    chosen = torch.full((t, kh, top), -1, dtype=torch.int32, device=dev)
    out = torch.empty(t, kh, g, d, device=dev)
    q = _rotate(x["q"]).reshape(t, kh, g, d) * d ** -0.5
    heads_at = torch.arange(kh, device=dev)[None, :, None]
    step = max(1, int(2.5e8 / (kh * d * max(width, top * page))))
    for t0 in range(0, t, step):
        part = slice(t0, min(t, t0 + step))
        table = x["table"].long()[x["seq"][part].long()].clamp(min=0)                      # [token][page]
        dots = torch.matmul(pool.block_codes[table].permute(0, 2, 1, 3), code[part, :, :, None]).squeeze(-1)      # whole numbers below 2^24
        score = dots * pool.block_scales[table].squeeze(-1).transpose(1, 2)
        n = pages[part, None, None]
        forced = (at < case["sinks"]) | (at >= n - case["local"])
        score = torch.where(forced, math.inf, score).masked_fill(at >= n, -math.inf)
        best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
        best = torch.sort(torch.where(torch.arange(best.shape[-1], device=dev) < n, best, width), -1).values
        ids = torch.where(best < width, best, -1)
        chosen[part, :, :ids.shape[-1]] = ids.int()
        at_rows = torch.arange(page, device=dev)
        own_page = torch.gather(table[:, None].expand(-1, kh, -1), 2, ids.clamp(min=0))
        slots = (own_page[..., None] * page + at_rows).flatten(2)
        seen = ((ids[..., None] * page + at_rows < x["lens"][part, None, None, None]) & (ids[..., None] >= 0)).flatten(2)
        k, v = ((pool.codes[i][slots, heads_at].float().reshape(*slots.shape, pool.groups, -1) * pool.scales[i][slots, heads_at][..., None]).flatten(-2) for i in range(2))
        s = torch.matmul(q[part], k.transpose(2, 3)).masked_fill(~seen[:, :, None], -math.inf)
        out[part] = _softmax_sum(s, v)
    return dict(chosen=chosen, out=_rotate_back(out).reshape(t, kh * g, d).to(x["q"].dtype))


# ------------------------------------------------------------------------------------------------ states and passes
_CTX = []


def _context():
    """The process's context, its calls ordered on torch's current stream (the default stream's handle is 0, its other name 1)."""
    import kronos_2t_b200 as k2
    if not _CTX:
        _CTX.append(k2.Context(0))
    _CTX[0].set_stream(torch.cuda.current_stream().cuda_stream or 1)
    return _CTX[0]


def prepare(case, seed):
    x = _inputs(case, seed)
    state = dict(case=case, x=x)
    block_keys = case["kind"] == "sparse" or case.get("block_keys", False)
    n = x["slots"].numel()
    if own:
        from kronos_2t_b200 import KvPool
        ctx = _context()
        pool = state["pool"] = KvPool(ctx, case["kv_heads"], case["head_dim"], case["bits"], case["page"], x["num_pages"], block_keys=block_keys)
        if case["kind"] == "cache":
            state["back"] = [torch.empty(n, case["kv_heads"], case["head_dim"], device="cuda") for _ in range(2)]
        else:
            pool.store_dev(case["dtype"], x["k"].data_ptr(), x["v"].data_ptr(), x["slots"].data_ptr(), n)
            state["out"] = torch.empty_like(x["q"])
            size = pool.workspace_bytes(case["heads"], x["q"].shape[0], case.get("prefix", 0))
            state["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
            if case["kind"] == "sparse":
                state["chosen"] = torch.empty(x["q"].shape[0], case["kv_heads"], case["top"], dtype=torch.int32, device="cuda")
    else:
        pool = state["pool"] = _Plain(case, x["num_pages"])
        if case["kind"] != "cache":
            for i in range(0, n, 65536):
                pool.store(x["slots"][i:i + 65536], x["k"][i:i + 65536], x["v"][i:i + 65536])
            if block_keys:
                pool.store_block_keys(x["num_pages"])
    if case["kind"] != "cache":
        del x["k"], x["v"]
    return state


def _run_own(state):
    case, x, pool = state["case"], state["x"], state["pool"]
    _context()
    if case["kind"] == "cache":
        n, back = case["n_tok"], state["back"]
        pool.store_dev(case["dtype"], x["k"].data_ptr(), x["v"].data_ptr(), x["slots"].data_ptr(), n)
        pool.load_dev("f32", x["slots"].data_ptr(), n, back[0].data_ptr(), back[1].data_ptr())
        return dict(k=back[0], v=back[1])
    t, work = x["q"].shape[0], (state["work"].data_ptr(), state["work"].numel())
    tokens = dict(dtype=case["dtype"], heads=case["heads"], n_tok=t, d_q=x["q"].data_ptr(), d_lens=x["lens"].data_ptr(), d_pages=x["table"].data_ptr(),
                  pages_stride=x["table"].shape[1], d_seq=x["seq"].data_ptr(), workspace=work)
    if case["kind"] == "prefix":
        pool.attend_dev(**tokens, d_out=state["out"].data_ptr(), d_prefix_pages=x["prefix_pages"].data_ptr(), prefix_len=case["prefix"])
        return state["out"]
    pool.select_dev(**tokens, top=case["top"], sinks=case["sinks"], local=case["local"], d_chosen=state["chosen"].data_ptr())
    pool.attend_chosen_dev(**tokens, top=case["top"], d_chosen=state["chosen"].data_ptr(), d_out=state["out"].data_ptr())
    return dict(chosen=state["chosen"], out=state["out"])


def run(state):
    if own:
        return _run_own(state)
    case, x, pool = state["case"], state["x"], state["pool"]
    if case["kind"] == "cache":
        pool.store(x["slots"], x["k"], x["v"])
        if case["block_keys"]:
            pool.store_block_keys(x["num_pages"])
        return dict(zip("kv", (_rotate_back(pool.rotated(i, x["slots"])) for i in range(2))))
    return (_plain_prefix if case["kind"] == "prefix" else _plain_sparse)(case, x, pool)


def work(case):
    kh, d, size = case["kv_heads"], case["head_dim"], 4 if case["dtype"] == "f32" else 2
    row = d + 4 if case["bits"] == 8 else d // 2 + d // 32
    if case["kind"] == "cache":
        n = case["n_tok"] * kh * 2
        return dict(bytes=n * (d * size + 2 * row + d * 4) + case["n_tok"] * 16, flops=n * d * 20)
    t, h, page = case["seqs"] * case["new"], case["heads"], case["page"]
    ends = 2 * t * h * d * size
    if case["kind"] == "prefix":         # own lengths spread evenly up to the longest
        mean = (case["new"] + case["own"]) / 2
        return dict(bytes=int(2 * row * kh * (case["prefix"] + case["seqs"] * mean) + ends), flops=int(4 * t * h * d * (case["prefix"] + mean)))
    mean = case["ctx"] * 0.55 if case["seqs"] > 1 else case["ctx"]
    seen = min(case["top"] * page, mean)
    pages = case["seqs"] * mean / page
    # every block key once; of the rows those that are chosen by a token, each at most once
    rows = min(case["seqs"] * mean, t * seen)
    return dict(bytes=int(pages * kh * (d + 4) + 2 * row * kh * rows + ends + 4 * t * kh * case["top"]),
                flops=int(4 * t * h * d * seen + 2 * t * kh * d * mean / page))


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_rotation(d):
    """The signed transform of a row as a matrix in 64 bits: r = x @ M, and x = r @ M.T."""
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < 64:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return (torch.block_diag(*[h / 8] * (d // 64)).cuda() * _signs(d).double()[:, None]).contiguous()


def _exact_transform(x):
    """The transform that the stored codes are defined by: fp32 sums, halves before their sum and difference."""
    if x.shape[-1] == 1:
        return x
    half = x.shape[-1] // 2
    a, b = _exact_transform(x[..., :half]), _exact_transform(x[..., half:])
    return torch.cat((a + b, a - b), -1)


def _exact_codes(r, bits):
    """Codes and scales of transformed rows, by their definition: quotients in 64 bits rounded to 32 (twice the digits and two more
    make that the quotient's own rounding), products likewise."""
    single = lambda y: y.float().double()
    r = r.double()
    if bits == 8:
        top = r.abs().amax(-1, keepdim=True)
        code = torch.round(single(r * single(127.0 / top)))
        nothing = top <= 2.0 ** -23
        return torch.where(nothing, 0.0, code), torch.where(nothing, 0.0, single(top / 127.0))
    centroids = torch.tensor(_CENTROIDS[8:], dtype=torch.float64, device=r.device)
    edges = torch.tensor(_EDGES, dtype=torch.float64, device=r.device)
    near = lambda y: torch.where(y >= 0, 1.0, -1.0) * centroids[torch.bucketize(y.abs(), edges, right=True)]
    r = r.unflatten(-1, (-1, 64))
    top = r.abs().amax(-1, keepdim=True)
    c = near(single(r * single(127.0 / top)))
    rc, num = single(r * c), 0.0
    for i in range(64):
        num = single(num + rc[..., i])
    fit = torch.where(num > 0, single(num / (c * c).sum(-1)), single(top.squeeze(-1) / 127.0))
    scale = fit.float().bfloat16().double()[..., None]
    return near(single(r * single(1.0 / scale))).flatten(-2), scale.squeeze(-1)


def _exact_rows(x, bits):
    """Stored rows in 64 bits, still transformed."""
    parts = (x.float() * _signs(x.shape[-1]) * 0.125).unflatten(-1, (-1, 64))
    code, scale = _exact_codes(_exact_transform(parts).flatten(-2), bits)
    return (code.unflatten(-1, (scale.shape[-1], -1)) * scale[..., None]).flatten(-2)


def exact(case, seed):
    x = _inputs(case, seed)
    kh, d, page, bits = case["kv_heads"], case["head_dim"], case["page"], case["bits"]
    turn = _exact_rotation(d)
    if case["kind"] == "cache":
        return {name: _exact_rows(x[name], bits) @ turn.T for name in ("k", "v")}
    cut = range(0, x["slots"].numel(), 65536)
    k, v = (torch.cat([_exact_rows(x[name][i:i + 65536], bits) for i in cut]) for name in ("k", "v"))       # in the order of writing
    t, g, new = x["q"].shape[0], case["heads"] // kh, case["new"]
    q = (x["q"].double() @ turn).reshape(t, kh, g, d) * d ** -0.5
    out = torch.empty(t, kh, g, d, dtype=torch.float64, device="cuda")
    lens, first = x["lens"].tolist(), case.get("prefix", 0)
    # rows of a sequence follow one another behind the prefix's
    ends = [lens[(b + 1) * new - 1] for b in range(case["seqs"])]
    starts = [first + sum(ends[:b]) for b in range(case["seqs"])]

    def attend(query, keys, values):
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", query, keys), -1)
        return torch.einsum("hgn,nhd->hgd", p, values)

    if case["kind"] == "prefix":
        at = torch.arange(first, device="cuda")
        for i in range(t):
            mine = torch.arange(starts[i // new], starts[i // new] + lens[i], device="cuda")
            rows = torch.cat((at, mine))
            out[i] = attend(q[i], k[rows], v[rows])
        return out.reshape(t, kh * g, d) @ turn.T
    # block keys of whole pages, the groups' queries, and the choice, in the arithmetic that defines them
    chosen = torch.full((t, kh, case["top"]), -1, dtype=torch.int32, device="cuda")
    keys_of = {}
    for b in range(case["seqs"]):
        whole = ends[b] // page
        rows = k[starts[b]:starts[b] + whole * page].float().reshape(whole, page, kh, d)
        total = torch.zeros(whole, kh, d, device="cuda")
        for i in range(page):
            total += rows[:, i]
        keys_of[b] = _exact_codes(total / page, 8) if whole else None
    group = x["q"].float().reshape(t, kh, g, d)
    query = group[:, :, 0].clone()
    for i in range(1, g):
        query += group[:, :, i]
    signed = (query * _signs(d) * 0.125).unflatten(-1, (-1, 64))
    query, _ = _exact_codes(_exact_transform(signed).flatten(-2), 8)
    for i in range(t):
        b, n = i // new, (lens[i] + page - 1) // page
        kept = sorted(set(range(min(case["sinks"], n))) | set(range(max(0, n - case["local"]), n)))
        free = torch.ones(n, dtype=torch.bool, device="cuda")
        free[kept] = False
        ids = torch.tensor(kept, device="cuda")[None].expand(kh, -1)
        want = min(case["top"], n) - len(kept)
        if want > 0:
            open_ids = free.nonzero().squeeze(1)
            code, scale = keys_of[b]
            dots = torch.einsum("hd,phd->hp", query[i], code[open_ids])
            score = (dots * scale[open_ids].squeeze(-1).T).float()
            best = torch.argsort(-score, dim=-1, stable=True)[:, :want]
            ids = torch.cat((ids, open_ids[best]), -1)
        ids = ids.sort(-1).values[:, :case["top"]]
        chosen[i, :, :ids.shape[1]] = ids.int()
        rows = (ids[..., None] * page + torch.arange(page, device="cuda")).flatten(1)       # [kv head][row]
        for h in range(kh):
            r = starts[b] + rows[h][rows[h] < lens[i]]
            out[i, h] = torch.softmax(q[i, h] @ k[r, h].T, -1) @ v[r, h]
    return dict(chosen=chosen, out=out.reshape(t, kh * g, d) @ turn.T)
