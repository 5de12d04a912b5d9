"""The attention-layer operators around the paged KV cache, as measured work.

Five operators of one serving step, in the order a step runs them:

  tables   block tables, positions and slot maps from the requests' lengths
  rope     per-head RMS norm of queries and keys with the rotary position
  append   the same, with the keys and values stored into the paged cache
  decode   one new token per sequence over a sliding window and a few first
           tokens that stay visible (sinks), read from the paged cache
  extend   the new tokens of a ragged batch under the same rule (prefill)

`listed()` names the cases, `draw()` makes more of the same ranges,
`prepare()` makes a case's inputs, `run()` is one pass, `work()` what a pass
cannot do without, and `exact()` the result in 64 bits.  With `own` false a
pass is plain torch arithmetic in 32 bits, with `own` true the framework's
entry points.
"""

import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"


def _mk():
    path = os.path.join(ROOT, "sglang-mlx_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from sglang_mlx_b200 import metal_kernels

    return metal_kernels


# ---- cases -------------------------------------------------------------------


def listed():
    return [
        # a decode step of a small server: every request adds one token; latency counts
        {"name": "tables_decode_64", "op": "tables", "kind": "decode", "seqs": 64, "longest": 4096, "block": 16},
        # a mixed continuous batch: 16 prefill chunks of 512 tokens beside 512 decodes
        {"name": "tables_mixed_528", "op": "tables", "kind": "mixed", "seqs": 528, "longest": 32768, "block": 32},
        # a batch of 256 prompts admitted at once, about 590 thousand tokens
        {"name": "tables_admit_256", "op": "tables", "kind": "admit", "seqs": 256, "longest": 4096, "block": 16},
        # queries and keys of a 256-sequence decode step, normed and rotated
        {"name": "rope_decode_256", "op": "rope", "tokens": 256, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "pairs": "half", "norm": True, "dtype": "bf16", "fused": True},
        # a prefill of 8192 tokens, interleaved pairs over half of each head, without norms
        {"name": "rope_prefill_8192", "op": "rope", "tokens": 8192, "heads": 28, "kv_heads": 4, "dim": 128, "rot": 64,
         "pairs": "interleaved", "norm": False, "dtype": "f16", "fused": True},
        # the same decode step with its keys and values stored, one token in each of 256 blocks
        {"name": "append_decode_256", "op": "append", "kind": "decode", "tokens": 256, "heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 128, "pairs": "half", "norm": True, "dtype": "bf16", "fused": True, "block": 16,
         "layout": "paged"},
        # 8192 prefill tokens stored in runs of whole blocks
        {"name": "append_prefill_8192", "op": "append", "kind": "prefill", "tokens": 8192, "heads": 28, "kv_heads": 4,
         "dim": 128, "rot": 128, "pairs": "half", "norm": True, "dtype": "bf16", "fused": True, "block": 32,
         "layout": "paged"},
        # one conversation of 131072 tokens: the latency of one long sequence
        {"name": "decode_1_w4096", "op": "decode", "seqs": 1, "lengths": "equal", "longest": 131072, "heads": 64,
         "kv_heads": 8, "dim": 128, "block": 32, "layout": "paged", "window": 4096, "sinks": 4, "dtype": "bf16"},
        # 256 sequences of 512 to 4096 tokens, most of them past the window
        {"name": "decode_256_w1024", "op": "decode", "seqs": 256, "lengths": "uniform", "longest": 4096, "heads": 32,
         "kv_heads": 8, "dim": 128, "block": 16, "layout": "paged", "window": 1024, "sinks": 4, "dtype": "bf16"},
        # 512 sequences of lognormal length on the token-major cache, an odd window and number of sinks
        {"name": "decode_512_w2047", "op": "decode", "seqs": 512, "lengths": "lognormal", "longest": 32768,
         "heads": 28, "kv_heads": 4, "dim": 128, "block": 32, "layout": "flash", "window": 2047, "sinks": 17,
         "dtype": "f16"},
        # short extends of a few sequences (a chat turn of 33 tokens), small heads
        {"name": "extend_4x33_w256", "op": "extend", "seqs": 4, "new": 33, "lengths": "uniform", "longest": 2048,
         "heads": 8, "kv_heads": 4, "dim": 64, "block": 16, "layout": "paged", "window": 256, "sinks": 4,
         "dtype": "bf16"},
        # 16 prefill chunks of 512 tokens over lognormal prefixes
        {"name": "extend_16x512_w1024", "op": "extend", "seqs": 16, "new": 512, "lengths": "lognormal",
         "longest": 32768, "heads": 28, "kv_heads": 4, "dim": 128, "block": 32, "layout": "paged", "window": 1024,
         "sinks": 4, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    n = int(round(lo * (hi / lo) ** rng.random()))
    return n + 1 if n == 3072 else max(lo, min(hi, n))


HEADS = [(32, 8), (64, 8), (28, 4), (8, 8), (16, 2), (5, 1), (8, 1)]


def draw(rng):
    op = rng.choice(["tables", "rope", "append", "decode", "extend"])
    if op == "tables":
        kind = rng.choice(["decode", "mixed", "admit"])
        return {"op": op, "kind": kind, "seqs": _log(rng, 1, 250 if kind == "admit" else 2000),
                "longest": _log(rng, 40, 4000), "block": rng.choice([8, 16, 32])}
    heads, kv_heads = rng.choice(HEADS)
    if op in ("rope", "append"):
        dim = rng.choice([64, 128, 128, 80, 96, 256])
        c = {"op": op, "tokens": _log(rng, 1, 4000), "heads": heads, "kv_heads": kv_heads, "dim": dim,
             "rot": rng.choice([dim, dim, dim // 2]), "pairs": rng.choice(["half", "interleaved"]),
             "norm": rng.random() < 0.6, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
             "fused": rng.random() < 0.7}
        if op == "append":
            c.update(kind=rng.choice(["decode", "prefill"]), block=rng.choice([8, 16, 32]),
                     layout=rng.choice(["paged", "paged", "flash", "pool"]))
            if c["layout"] == "pool":
                c["block"] = 1
        return c
    layout = rng.choice(["paged", "paged", "flash", "pool"])
    c = {"op": op, "lengths": rng.choice(["uniform", "lognormal", "equal"]), "heads": heads, "kv_heads": kv_heads,
         "dim": rng.choice([64, 128]), "block": 1 if layout == "pool" else rng.choice([8, 16, 32]), "layout": layout,
         "window": _log(rng, 16, 4096), "sinks": rng.choice([0, 1, 4, 17, 64]),
         "dtype": rng.choice(["bf16", "f16"])}
    if op == "decode":
        c.update(seqs=_log(rng, 1, 250), longest=_log(rng, 30, 9000))
    else:
        c.update(seqs=_log(rng, 1, 8), new=_log(rng, 1, 500), longest=_log(rng, 600, 9000))
    return c


# ---- inputs ------------------------------------------------------------------


def _lengths(kind, n, longest, rs):
    """Cached tokens of n sequences: equal, uniform from an eighth of the longest, or lognormal (median 1500)."""
    if kind == "equal":
        return np.full(n, longest, np.int64)
    if kind == "uniform":
        return rs.randint(max(1, longest // 8), longest + 1, n).astype(np.int64)
    return np.clip(np.round(np.exp(np.log(1500.0) + rs.randn(n))), min(16, longest), longest).astype(np.int64)


def _ints(a, dtype=torch.int32):
    return torch.as_tensor(np.ascontiguousarray(a)).to(DEV, dtype)


def _tables(lens, block, gen, spare=3):
    """Block tables over a seeded permutation of the pool, and the pool's block count."""
    need = -(-lens // block)
    width = int(need.max()) if len(need) else 1
    total = int(need.sum())
    blocks = total + spare
    order = torch.randperm(blocks, generator=gen, device=DEV, dtype=torch.int64)
    first = _ints(np.concatenate([[0], np.cumsum(need)[:-1]]), torch.int64)
    j = torch.arange(width, device=DEV)
    inside = j[None, :] < _ints(need, torch.int64)[:, None]
    at = (first[:, None] + j[None, :]).clamp(max=blocks - 1)
    return torch.where(inside, order[at], -1).to(torch.int32).contiguous(), blocks


def _cache_shapes(layout, blocks, block, kv_heads, dim, itemsize):
    x = 16 // itemsize
    if layout == "paged":
        return (blocks, kv_heads, dim // x, block, x), (blocks, kv_heads, dim, block)
    if layout == "flash":
        return ((blocks, block, kv_heads, dim),) * 2
    return ((blocks, kv_heads, dim),) * 2


def _caches(c, blocks, gen, dtype):
    ks, vs = _cache_shapes(c["layout"], blocks, c["block"], c["kv_heads"], c["dim"], dtype.itemsize)
    return (torch.randn(ks, generator=gen, device=DEV, dtype=dtype),
            torch.randn(vs, generator=gen, device=DEV, dtype=dtype))


def _new_tokens(c, rs):
    """New tokens of each request: their sum goes by the case alone, their order by `rs`."""
    n, longest, fixed = c["seqs"], c["longest"], np.random.RandomState(7)
    if c["op"] == "decode" or c.get("kind") == "decode":
        return np.ones(n, np.int64)
    if c["op"] == "extend":  # ragged: one chunk whole, the others from a half up
        new = fixed.randint(max(1, c["new"] // 2), c["new"] + 1, n)
        new[0] = c["new"]
    elif c["kind"] == "admit":
        new = _lengths("uniform", n, longest, fixed)
    else:  # one request in 33 brings a chunk, the others one token
        new = np.where(np.arange(n) < max(1, n // 33), min(512, max(1, longest // 8)), 1)
    return rs.permutation(new.astype(np.int64))


def _tables_lengths(c, rs):
    """(cached tokens, new tokens) of each request of a tables case."""
    new = _new_tokens(c, rs)
    if c["kind"] == "admit":
        return np.zeros(c["seqs"], np.int64), new
    return _lengths("uniform" if c["kind"] == "decode" else "lognormal", c["seqs"], c["longest"], rs), new


def prepare(case, seed):
    c = case
    rs = np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = {"op": c["op"], "case": c}
    if c["op"] == "tables":
        prefix, new = _tables_lengths(c, rs)
        block = c["block"]
        have = -(-prefix // block)
        need = -(-(prefix + new) // block)
        tables, used = _tables(prefix, block, gen, spare=int((need - have).sum()) + 8)
        width = -(-(c["longest"] + 512) // block) + 2  # the table has room for the longest request
        wide = torch.full((len(prefix), width), -1, dtype=torch.int32, device=DEV)
        wide[:, : tables.shape[1]] = tables
        # the pool's other blocks are free, in an order of their own
        taken = torch.zeros(used, dtype=torch.bool, device=DEV)
        taken[tables[tables >= 0].long()] = True
        free = torch.nonzero(~taken).flatten().to(torch.int32)
        s.update(tables=wide, prefix=_ints(prefix), new=_ints(new),
                 free=free[torch.randperm(free.numel(), generator=gen, device=DEV)].contiguous(),
                 tokens=int(new.sum()), block=block)
        n, t = len(prefix), s["tokens"]
        s.update(kv_lens=torch.empty(n, dtype=torch.int32, device=DEV),
                 qo_indptr=torch.empty(n + 1, dtype=torch.int32, device=DEV),
                 positions=torch.empty(t, dtype=torch.int32, device=DEV),
                 slots=torch.empty(t, dtype=torch.int64, device=DEV),
                 used=torch.empty(1, dtype=torch.int32, device=DEV))
        return s
    dtype = DTYPES[c["dtype"]]
    if c["op"] in ("rope", "append"):
        t, h, hk, d = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        if c["fused"]:  # slices of one projection's output
            qkv = torch.randn((t, h + 2 * hk, d), generator=gen, device=DEV, dtype=dtype)
            q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        else:
            q, k, v = (torch.randn((t, n, d), generator=gen, device=DEV, dtype=dtype) for n in (h, hk, hk))
        longest = 32768
        # the angles in 64 bits, the table in 32
        freq = 10000.0 ** (-np.arange(0, c["rot"], 2, dtype=np.float64) / c["rot"])
        ang = torch.arange(longest, device=DEV, dtype=torch.float64)[:, None] * torch.as_tensor(freq, device=DEV)
        s.update(q=q, k=k, v=v, table=torch.cat([ang.cos(), ang.sin()], 1).float(),
                 q_out=torch.empty((t, h, d), dtype=dtype, device=DEV),
                 positions=torch.randint(0, longest, (t,), generator=gen, device=DEV, dtype=torch.int32))
        s["qw"] = 1 + 0.1 * torch.randn(d, generator=gen, device=DEV) if c["norm"] else None
        s["kw"] = 1 + 0.1 * torch.randn(d, generator=gen, device=DEV) if c["norm"] else None
        if c["norm"]:
            s["qw"], s["kw"] = s["qw"].to(dtype), s["kw"].to(dtype)
        if c["op"] == "rope":
            s["k_out"] = torch.empty((t, hk, d), dtype=dtype, device=DEV)
            return s
        block = c["block"]
        if c["kind"] == "decode":  # one token in a block of its own, at any offset
            blocks = t + 3
            slots = torch.randperm(blocks, generator=gen, device=DEV)[:t] * block
            slots = slots + torch.randint(0, block, (t,), generator=gen, device=DEV)
        else:  # runs of consecutive tokens through blocks in any order
            blocks = -(-t // block) + 3
            order = torch.randperm(blocks, generator=gen, device=DEV)
            i = torch.arange(t, device=DEV)
            slots = order[i // block] * block + i % block
            s["positions"] = (i + int(rs.randint(0, longest - t))).to(torch.int32)
        s["slots"] = slots.to(torch.int64)
        s["kc"], s["vc"] = _caches(c, blocks, gen, dtype)
        return s
    n = c["seqs"]
    new = _new_tokens(c, rs)
    lens = np.maximum(_lengths(c["lengths"], n, c["longest"], rs), new)
    tables, blocks = _tables(lens, c["block"], gen)
    kc, vc = _caches(c, blocks, gen, dtype)
    rows = int(new.sum())
    s.update(tables=tables, kc=kc, vc=vc, lens=_ints(lens), scale=c["dim"] ** -0.5, longest=int(lens.max()),
             q=torch.randn((rows, c["heads"], c["dim"]), generator=gen, device=DEV, dtype=dtype),
             out=torch.empty((rows, c["heads"], c["dim"]), dtype=dtype, device=DEV), new_most=int(new.max()),
             indptr=_ints(np.concatenate([[0], np.cumsum(new)])))
    return s


# ---- one pass ----------------------------------------------------------------


def run(state):
    s, c = state, state["case"]
    return {"tables": _run_tables, "rope": _run_rope, "append": _run_append, "decode": _run_decode,
            "extend": _run_extend}[s["op"]](s, c)


def _run_tables(s, c):
    if own:
        _mk().build_step_tables(s["tables"], s["prefix"], s["new"], s["free"], s["block"], kv_lens=s["kv_lens"],
                                qo_indptr=s["qo_indptr"], positions=s["positions"], slot_mapping=s["slots"],
                                blocks_used=s["used"])
        return s["tables"], s["kv_lens"], s["qo_indptr"], s["positions"], s["slots"], s["used"]
    prefix, new, block = s["prefix"].long(), s["new"].long(), s["block"]
    total = prefix + new
    first = (prefix + block - 1) // block
    count = (total + block - 1) // block - first
    ends, taken = new.cumsum(0), count.cumsum(0)
    j = torch.arange(s["tables"].shape[1], device=DEV)[None, :] - first[:, None]
    inside = (j >= 0) & (j < count[:, None])
    at = (taken - count)[:, None] + j
    tables = torch.where(inside, s["free"][at.clamp(0, s["free"].numel() - 1)], s["tables"])
    i = torch.arange(s["tokens"], device=DEV)
    seq = torch.bucketize(i, ends, right=True)
    pos = prefix[seq] + i - (ends - new)[seq]
    slots = tables[seq, pos // block].long() * block + pos % block
    indptr = torch.cat([ends.new_zeros(1), ends])
    return tables, total.int(), indptr.int(), pos.int(), slots, taken[-1:].int()


def _rotated(x, weight, table, positions, c):
    """x in 32 bits, normed over each head and rotated by its position's angles."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    cs = table[positions.long()]
    half = c["rot"] // 2
    cos, sin = cs[:, None, :half], cs[:, None, half:]
    y, rest = x[..., :c["rot"]], x[..., c["rot"]:]
    if c["pairs"] == "half":
        a, b = y[..., :half], y[..., half:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, rest], -1)


def _run_rope(s, c):
    if own:
        _mk().qk_norm_rope(s["q"], s["k"], s["positions"], s["table"], q_weight=s["qw"], k_weight=s["kw"], eps=1e-6,
                           interleaved=c["pairs"] == "interleaved", q_out=s["q_out"], k_out=s["k_out"])
        return s["q_out"], s["k_out"]
    return (_rotated(s["q"], s["qw"], s["table"], s["positions"], c).to(s["q"].dtype),
            _rotated(s["k"], s["kw"], s["table"], s["positions"], c).to(s["k"].dtype))


def _run_append(s, c):
    if own:
        _mk().qk_norm_rope_append(s["q"], s["k"], s["v"], s["positions"], s["table"], s["kc"], s["vc"], s["slots"],
                                  q_weight=s["qw"], k_weight=s["kw"], eps=1e-6,
                                  interleaved=c["pairs"] == "interleaved", q_out=s["q_out"])
        return s["q_out"], s["kc"], s["vc"]
    q = _rotated(s["q"], s["qw"], s["table"], s["positions"], c).to(s["q"].dtype)
    k = _rotated(s["k"], s["kw"], s["table"], s["positions"], c).to(s["k"].dtype)
    blk, off = s["slots"] // c["block"], s["slots"] % c["block"]
    kc, vc = s["kc"], s["vc"]
    if c["layout"] == "paged":
        kc[blk, :, :, off] = k.view(k.shape[0], k.shape[1], -1, kc.shape[-1])
        vc[blk, :, :, off] = s["v"]
    elif c["layout"] == "flash":
        kc[blk, off] = k
        vc[blk, off] = s["v"]
    else:
        kc[blk] = k
        vc[blk] = s["v"]
    return q, kc, vc


def _gathered(s, c, pos):
    """K and V in 32 bits, [sequences, positions, kv heads, dim], at the given positions of each sequence."""
    blk = torch.gather(s["tables"].long(), 1, pos // c["block"])
    off = pos % c["block"]
    n, m = pos.shape
    if c["layout"] == "paged":
        k, v = s["kc"][blk, :, :, off].reshape(n, m, c["kv_heads"], c["dim"]), s["vc"][blk, :, :, off]
    elif c["layout"] == "flash":
        k, v = s["kc"][blk, off], s["vc"][blk, off]
    else:
        k, v = s["kc"][blk], s["vc"][blk]
    return k.float(), v.float()


def _attended(q, k, v, seen, scale):
    """softmax(scale q k) v over the seen positions: q [n, kv heads, rows, dim], seen [n, 1, rows, positions]."""
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * scale
    x = torch.where(seen, x, float("-inf"))
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == float("-inf"), 0.0, top))
    return torch.matmul(e, v.permute(0, 2, 1, 3)) / (e.sum(-1, keepdim=True) + 1e-6)


def _run_decode(s, c):
    if own:
        _mk().paged_attention_window(s["q"], s["kc"], s["vc"], s["tables"], s["lens"], c["kv_heads"], s["scale"],
                                     c["block"], s["longest"], c["window"], c["sinks"], out=s["out"])
        return s["out"]
    ln = s["lens"].long()[:, None]
    sink = torch.arange(c["sinks"], device=DEV)[None, :].expand(ln.shape[0], -1)
    win = ln - c["window"] + torch.arange(c["window"], device=DEV)[None, :]
    pos = torch.cat([sink, win], 1)
    seen = torch.cat([sink < ln, win >= c["sinks"]], 1)
    k, v = _gathered(s, c, torch.where(seen, pos, 0))
    q = s["q"].float().view(ln.shape[0], c["kv_heads"], -1, c["dim"])
    o = _attended(q, k, v, seen[:, None, None, :], s["scale"])
    return o.reshape(s["q"].shape).to(s["q"].dtype)


def _run_extend(s, c):
    if own:
        _mk().paged_prefill_window(s["q"], s["kc"], s["vc"], s["tables"], s["indptr"], s["lens"], c["kv_heads"],
                                   s["scale"], c["block"], c["window"], c["sinks"], max_q_len=s["new_most"],
                                   out=s["out"])
        return s["out"]
    starts, ends = s["indptr"][:-1].long(), s["indptr"][1:].long()
    ln = s["lens"].long()
    prefix = ln - (ends - starts)
    n, most, g = ln.numel(), s["new_most"], c["heads"] // c["kv_heads"]
    t = torch.arange(most, device=DEV)
    rows = (starts[:, None] + t[None, :]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[rows].view(n, most, c["kv_heads"], g, c["dim"]).permute(0, 2, 1, 3, 4)
    sink = torch.arange(c["sinks"], device=DEV)[None, :].expand(n, -1)
    win = (prefix - c["window"] + 1)[:, None] + torch.arange(c["window"] + most - 1, device=DEV)[None, :]
    pos = torch.cat([sink, win], 1)
    there = torch.cat([sink < ln[:, None], (win >= c["sinks"]) & (win < ln[:, None])], 1)
    k, v = _gathered(s, c, torch.where(there, pos, 0))
    at = (prefix[:, None] + t[None, :])[:, :, None]
    seen = there[:, None, :] & (pos[:, None, :] <= at)
    seen = seen & ((pos[:, None, :] > at - c["window"]) | (pos[:, None, :] < c["sinks"]))
    seen = seen[:, None, :, None, :].expand(-1, -1, -1, g, -1).reshape(n, 1, most * g, -1)
    o = _attended(q.reshape(n, c["kv_heads"], most * g, c["dim"]), k, v, seen, s["scale"])
    o = o.view(n, c["kv_heads"], most, g, c["dim"])
    i = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.bucketize(i, ends, right=True)
    return o[seq, :, i - starts[seq]].reshape(s["q"].shape).to(s["q"].dtype)


# ---- what a pass cannot do without -------------------------------------------


def work(case):
    c = case
    rs = np.random.RandomState(1)
    if c["op"] == "tables":
        prefix, new = _tables_lengths(c, rs)
        blocks = int((-(-(prefix + new) // c["block"]) + -prefix // c["block"]).sum())
        # lengths in; lengths, offsets, positions (4 bytes) and slots (8) out; each new block's id in and out
        return {"bytes": len(prefix) * 16 + int(new.sum()) * 12 + blocks * 8, "flops": 4 * int(new.sum())}
    size = DTYPES[c["dtype"]].itemsize
    if c["op"] in ("rope", "append"):
        rows = c["heads"] + c["kv_heads"] * (2 if c["op"] == "append" else 1)
        per_token = 2 * rows * c["dim"] * size + 4 + 4 * c["rot"] + (8 if c["op"] == "append" else 0)
        return {"bytes": c["tokens"] * per_token,
                "flops": c["tokens"] * (c["heads"] + c["kv_heads"]) * (3 * c["rot"] + (4 * c["dim"] if c["norm"] else 0))}
    n = c["seqs"]
    new = _new_tokens(c, rs)
    lens = np.maximum(_lengths(c["lengths"], n, c["longest"], rs), new)
    prefix = lens - new
    # distinct cache tokens that some new token sees, and (new token, seen token) pairs
    first = np.maximum(prefix + 1 - c["window"], 0)
    tokens = int((lens - first + np.minimum(c["sinks"], first)).sum())
    pairs = 0
    for p, m in zip(prefix, new):
        i = np.arange(p, p + m)
        start = np.maximum(i + 1 - c["window"], 0)
        pairs += int((i + 1 - start + np.minimum(c["sinks"], start)).sum())
    return {"bytes": 2 * tokens * c["kv_heads"] * c["dim"] * size + 2 * int(new.sum()) * c["heads"] * c["dim"] * size
            + 4 * tokens // c["block"] + 4 * n,
            "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---- the results in 64 bits --------------------------------------------------


def _exact_row_ops(x, weight, positions, c):
    """Norm and rotation of x [tokens, heads, dim] with complex numbers: each pair times e^(i angle)."""
    x = x.to(torch.float64)
    if weight is not None:
        x = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / c["dim"] + 1e-6)
        x = x * weight.to(torch.float64)
    half = c["rot"] // 2
    order = np.arange(c["rot"]).reshape(2, half).T if c["pairs"] == "half" else np.arange(c["rot"]).reshape(half, 2)
    first, second = (torch.as_tensor(np.ascontiguousarray(order[:, e]), device=x.device) for e in (0, 1))
    freq = torch.exp(-torch.arange(half, dtype=torch.float64, device=x.device) * (np.log(10000.0) / half))
    angle = positions.to(torch.float64)[:, None, None] * freq
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), angle)
    x[..., first], x[..., second] = z.real, z.imag
    return x


def exact(case, seed):
    c = case
    if c["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if c["op"] in ("rope", "append"):
        q = _exact_row_ops(s["q"], s["qw"], s["positions"], c)
        k = _exact_row_ops(s["k"], s["kw"], s["positions"], c)
        if c["op"] == "rope":
            return q, k
        kc, vc, v = s["kc"].double(), s["vc"].double(), s["v"].double()
        t = k.shape[0]
        if c["layout"] == "paged":  # element d of token i: block, head, chunk, offset, place in the chunk
            x = kc.shape[-1]
            blk, off = (s["slots"] // c["block"])[:, None, None], (s["slots"] % c["block"])[:, None, None]
            h = torch.arange(c["kv_heads"], device=DEV)[None, :, None]
            d = torch.arange(c["dim"], device=DEV)[None, None, :]
            kc[blk, h, d // x, off, d % x] = k
            vc[blk, h, d, off] = v
        else:
            kc.view(-1, c["kv_heads"], c["dim"]).index_copy_(0, s["slots"], k)
            vc.view(-1, c["kv_heads"], c["dim"]).index_copy_(0, s["slots"], v)
        assert t == v.shape[0]
        return q, kc, vc
    if work(case)["flops"] > 4e12:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    bounds, lens = s["indptr"].tolist(), s["lens"].tolist()
    g = c["heads"] // c["kv_heads"]
    for b, ln in enumerate(lens):
        lo, hi = bounds[b], bounds[b + 1]
        prefix = ln - (hi - lo)
        first = max(prefix + 1 - c["window"], 0)
        j = torch.cat([torch.arange(min(c["sinks"], first), device=DEV), torch.arange(first, ln, device=DEV)])
        ids = s["tables"][b][j // c["block"]].long()
        off = j % c["block"]
        if c["layout"] == "paged":
            k = s["kc"].permute(0, 3, 1, 2, 4)[ids, off].flatten(2).double()
            v = s["vc"].permute(0, 3, 1, 2)[ids, off].double()
        else:
            shape = (-1, c["kv_heads"], c["dim"])
            k = s["kc"].view(shape)[ids * c["block"] + off].double()
            v = s["vc"].view(shape)[ids * c["block"] + off].double()
        q = s["q"][lo:hi].double().view(hi - lo, c["kv_heads"], g, c["dim"])
        i = torch.arange(prefix, ln, device=DEV)[:, None]
        hidden = (j[None, :] > i) | ((j[None, :] <= i - c["window"]) & (j[None, :] >= c["sinks"]))
        logit = torch.einsum("thgd,jhd->thgj", q, k) * s["scale"]
        logit.masked_fill_(hidden[:, None, None, :], float("-inf"))
        # the denominator's 1e-6 belongs to the definition of the decode: relative to the largest term
        p = torch.exp(logit - logit.max(-1, keepdim=True).values)
        p = p / (p.sum(-1, keepdim=True) + 1e-6)
        out[lo:hi] = torch.einsum("thgj,jhd->thgd", p, v).reshape(hi - lo, c["heads"], c["dim"])
    return out
