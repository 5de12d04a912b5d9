"""Step tables, rotary tables, and the per-head norm with the rotary position
(alone and with the append), against plain NumPy in float64 / integers."""

import ctypes
import math
import os

import numpy as np
import pytest

from oracle import kv_oracle
from sglang_mlx_b200 import _lib, dlpack, dtypes
from sglang_mlx_b200 import metal_kernels as mk
from sglang_mlx_b200.device_array import DeviceArray, Stream

# ---- step tables ----------------------------------------------------------------


def plain_tables(tables, prefix, new, free, bs, capacity):
    t = tables.copy()
    at, slots, pos, indptr = 0, [], [], [0]
    for b, (p, n) in enumerate(zip(prefix, new)):
        first, last = -(-p // bs), -(-(p + n) // bs)
        t[b, first:last] = free[at:at + last - first]
        at += last - first
        for i in range(p, p + n):
            pos.append(i)
            slots.append(int(t[b, i // bs]) * bs + i % bs)
        indptr.append(indptr[-1] + n)
    pad = capacity - len(pos)
    return t, np.asarray(prefix) + new, indptr, pos + [-1] * pad, slots + [-1] * pad, at


def run_tables(tables, prefix, new, free, bs, capacity, slot_dtype="int64"):
    dev = lambda a, dt="int32": DeviceArray.from_numpy(np.asarray(a), dtype=dt)  # noqa: E731
    bt = dev(tables)
    out = mk.build_step_tables(bt, dev(np.asarray(prefix, np.int32)), dev(np.asarray(new, np.int32)),
                               dev(np.asarray(free, np.int32)), bs, capacity,
                               slot_mapping=DeviceArray.zeros((capacity,), slot_dtype))
    return [np.asarray(x.to_numpy()) for x in out]


def tables_case(seed, B, bs, longest, most_new):
    rng = np.random.default_rng(seed)
    prefix = rng.integers(0, longest + 1, B)
    new = rng.integers(0, most_new + 1, B)
    need, have = -(-(prefix + new) // bs), -(-prefix // bs)
    blocks = rng.permutation(int(need.sum()) + 4)
    tables = np.full((B, int(need.max(initial=0)) + 2), -7, np.int64)
    at = 0
    for b in range(B):
        tables[b, :have[b]] = blocks[at:at + have[b]]
        at += have[b]
    return tables, prefix, new, blocks[at:]


@pytest.mark.gpu
@pytest.mark.parametrize("B,bs,longest,most_new,extra", [
    (1, 16, 0, 1, 0), (1, 16, 100, 1, 3), (3, 8, 40, 50, 5), (64, 16, 4096, 1, 0), (65, 32, 50, 9, 1),
    (300, 1, 20, 6, 2), (1023, 16, 100, 3, 0), (1024, 16, 100, 3, 7), (1025, 7, 100, 3, 1), (4000, 16, 60, 5, 0),
    (5, 16, 10, 40000, 11), (2, 48, 0, 0, 4)])
@pytest.mark.parametrize("slot_dtype", ["int32", "int64"])
def test_step_tables(gpu, B, bs, longest, most_new, extra, slot_dtype):
    case = tables_case(B * 31 + bs, B, bs, longest, most_new)
    capacity = int(case[2].sum()) + extra
    want = plain_tables(*case, bs, capacity)
    got = run_tables(*case, bs, capacity, slot_dtype)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g.reshape(-1), np.asarray(w).reshape(-1))
    assert _lib.get_status(0, clear=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("B,bs,longest,most_new", [(1, 16, 100, 1), (64, 16, 4096, 1), (300, 16, 500, 40),
                                                   (1500, 16, 100, 3), (4000, 16, 60, 5), (5, 16, 10, 40000), (2, 16, 0, 0)])
@pytest.mark.parametrize("into", ["prefix_lens", "new_lens"])
def test_step_tables_update_lengths_in_place(gpu, B, bs, longest, most_new, into):
    """A server that keeps its lengths on the device passes them as the output too: everything else as without."""
    tables, prefix, new, free = tables_case(B * 37 + bs, B, bs, longest, most_new)
    if B > 2:
        new[1] = 0
    capacity = int(new.sum()) + 3
    want = plain_tables(tables, prefix, new, free, bs, capacity)
    dev = {n: DeviceArray.from_numpy(np.asarray(a), dtype="int32") for n, a in
           (("tables", tables), ("prefix_lens", prefix), ("new_lens", new), ("free", free))}
    got = mk.build_step_tables(dev["tables"], dev["prefix_lens"], dev["new_lens"], dev["free"], bs, capacity,
                               kv_lens=dev[into])
    assert got.kv_lens is dev[into]
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g.to_numpy().reshape(-1), np.asarray(w).reshape(-1))
    other = "new_lens" if into == "prefix_lens" else "prefix_lens"
    np.testing.assert_array_equal(dev[other].to_numpy(), new if other == "new_lens" else prefix)
    assert _lib.get_status(0, clear=True) == 0


@pytest.mark.gpu
def test_step_tables_in_place_reads_bad_lengths_as_zero(gpu):
    lens = DeviceArray.from_numpy(np.array([5, -3, 7, 2**31 - 5], np.int32))
    new = DeviceArray.from_numpy(np.array([1, 4, -2, 9], np.int32))
    tables = DeviceArray.from_numpy(np.full((4, 2), 1, np.int32))
    mk.build_step_tables(tables, lens, new, DeviceArray.from_numpy(np.array([3], np.int32)), 16, 1, kv_lens=lens)
    assert lens.to_numpy().tolist() == [6, 0, 0, 0]
    assert _lib.get_status(0, clear=True) == _lib.STATUS_INDEX_OOB


@pytest.mark.gpu
def test_step_tables_no_requests(gpu):
    got = run_tables(np.zeros((0, 4), np.int32), [], [], [1, 2], 16, 3)
    assert got[2].tolist() == [0] and got[3].tolist() == [-1] * 3 and got[4].tolist() == [-1] * 3
    assert got[5].tolist() == [0] and _lib.get_status(0, clear=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["free", "table", "capacity", "negative", "hole", "slot32"])
def test_step_tables_flags_what_does_not_fit(gpu, what):
    tables, prefix, new, free, bs, cap, sd = np.full((2, 4), -1, np.int64), [5, 0], [20, 30], [9, 8, 7], 16, 50, "int64"
    tables[0, 0] = 3
    if what == "free":  # needs 1 + 2 blocks, one is free
        free = [9]
        want = [-1] * 50
        want[:20] = [3 * 16 + i for i in range(5, 16)] + [9 * 16 + i for i in range(9)]
    elif what == "table":
        new = [20, 70]
        cap, free = 90, [9, 8, 7, 6, 5, 4]
        want = [3 * 16 + i for i in range(5, 16)] + [9 * 16 + i for i in range(9)]
        want += [b * 16 + i for b in (8, 7, 6, 5) for i in range(16)] + [-1] * 6
    elif what == "capacity":
        cap = 45
        want = ([3 * 16 + i for i in range(5, 16)] + [9 * 16 + i for i in range(9)] + [8 * 16 + i for i in range(16)] +
                [7 * 16 + i for i in range(14)])[:45]
    elif what == "negative":
        new = [-4, 30]
        want = [9 * 16 + i for i in range(16)] + [8 * 16 + i for i in range(14)] + [-1] * 20
    elif what == "hole":  # the block that the cached tokens end in is not in the table
        tables[0, 0] = -1
        want = [-1] * 11 + [9 * 16 + i for i in range(9)] + [8 * 16 + i for i in range(16)] + [7 * 16 + i for i in range(14)]
    else:
        sd, free = "int32", [1 << 27, 8, 7]  # block 2^27 of 16 tokens: past int32
        want = [3 * 16 + i for i in range(5, 16)] + [-1] * 9 + [8 * 16 + i for i in range(16)] + [7 * 16 + i for i in range(14)]
    got = run_tables(tables, prefix, new, free, bs, cap, sd)
    assert got[4].tolist() == want
    assert _lib.get_status(0, clear=True) == _lib.STATUS_INDEX_OOB


# ---- rotary frequencies and tables ------------------------------------------------


def test_rotary_frequencies():
    f, a = mk.rotary_frequencies(8, 10000.0)
    np.testing.assert_allclose(f, [1.0, 0.1, 0.01, 0.001], rtol=1e-14)
    assert a == 1.0
    np.testing.assert_allclose(mk.rotary_frequencies(8, 10000.0, {"type": "linear", "factor": 4.0})[0],
                               np.array([1.0, 0.1, 0.01, 0.001]) / 4, rtol=1e-14)
    # ntk: the highest frequency keeps, the lowest is divided by the factor
    n = mk.rotary_frequencies(128, 10000.0, {"type": "ntk", "factor": 8.0})[0]
    g = mk.rotary_frequencies(128, 10000.0)[0]
    assert n[0] == 1.0 and abs(n[-1] * 8.0 / g[-1] - 1) < 1e-12
    # bands: short wavelengths keep, long ones are divided, between them monotone
    b = mk.rotary_frequencies(128, 500000.0, {"type": "bands", "factor": 8.0, "original_max_position": 8192})[0]
    g = mk.rotary_frequencies(128, 500000.0)[0]
    turns = 8192 * g / (2 * math.pi)
    np.testing.assert_allclose(b[turns >= 4], g[turns >= 4], rtol=1e-14)
    np.testing.assert_allclose(b[turns <= 1], g[turns <= 1] / 8, rtol=1e-14)
    assert (np.diff(b) < 0).all()
    # yarn: as they are up to beta_fast turns, divided below beta_slow turns, the factor of the rotated part
    y, a = mk.rotary_frequencies(128, 10000.0, {"type": "yarn", "factor": 4.0, "original_max_position": 4096})
    g = mk.rotary_frequencies(128, 10000.0)[0]
    turns = 4096 * g / (2 * math.pi)
    np.testing.assert_allclose(y[turns > 33], g[turns > 33], rtol=1e-14)
    np.testing.assert_allclose(y[turns < 0.9], g[turns < 0.9] / 4, rtol=1e-14)
    assert abs(a - (0.1 * math.log(4.0) + 1.0)) < 1e-15


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0),
                                dict(rotary_dim=8, scaling={"type": "other"}),
                                dict(rotary_dim=8, scaling={"type": "linear", "factor": 0.0}),
                                dict(rotary_dim=8, scaling={"type": "bands", "factor": 2.0, "original_max_position": 64,
                                                            "low_freq_factor": 4.0, "high_freq_factor": 1.0})])
def test_rotary_frequencies_refusals(kw):
    with pytest.raises(ValueError):
        mk.rotary_frequencies(**kw)


def table64(positions, rot, base=10000.0, scaling=None):
    f, a = mk.rotary_frequencies(rot, base, scaling)
    ang = np.asarray(positions, np.float64)[:, None] * f
    return np.concatenate([np.cos(ang), np.sin(ang)], 1) * a


@pytest.mark.gpu
@pytest.mark.parametrize("rot,rows,scaling", [(2, 5, None), (64, 70000, None), (128, 4097, {"type": "yarn", "factor": 8.0,
                                               "original_max_position": 4096}), (256, 33, {"type": "ntk", "factor": 2.0})])
def test_rotary_table(gpu, rot, rows, scaling):
    t = mk.rotary_table(rows, rot, scaling=scaling).to_numpy()
    # one rounding to float32 of values up to 1.21: at most 2^-24 * 2 (and the 64-bit sine's own error)
    assert np.abs(t - table64(np.arange(rows), rot, scaling=scaling)).max() <= 1.2e-7


# ---- norm and rotation --------------------------------------------------------------


def plain_rope(x, w, cs, rot, interleaved, eps):
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    half = rot // 2
    c, s = cs[:, None, :half].astype(np.float64), cs[:, None, half:].astype(np.float64)
    out = x.copy()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :half], x[..., half:rot]
        out[..., :half], out[..., half:rot] = a * c - b * s, b * c + a * s
    return out


# half a step of the output's type (2^-9, 2^-12, 2^-25 of the value), doubled for a value whose 32-bit
# error moves it across a rounding boundary, and the 32-bit arithmetic's own error on values up to about 8
TOL = {"bfloat16": (1e-5, 2.0 ** -8), "float16": (1e-5, 2.0 ** -11), "float32": (1e-5, 2.0 ** -20)}


def close(got, want, dtype):
    atol, rtol = TOL[dtype]
    bad = np.abs(got - want) - (atol + rtol * np.abs(want))
    assert np.isfinite(got).all() and bad.max() <= 0, f"{dtype}: {np.abs(got - want).max():.3g}"


class Rope:
    def __init__(self, seed, dtype, T, hq, hkv, d, rot, norm, wdtype=None, fused=True, rows=5000, poison=False):
        rng = np.random.default_rng(seed)
        rnd = lambda *s: kv_oracle.round_to(rng.standard_normal(s).astype(np.float32), dtype)  # noqa: E731
        self.dtype, self.d, self.rot, self.hq, self.hkv, self.T = dtype, d, rot, hq, hkv, T
        wide = rnd(T, hq + 2 * hkv, d)
        self.q, self.k, self.v = wide[:, :hq], wide[:, hq:hq + hkv], wide[:, hq + hkv:]
        if fused:
            dev = DeviceArray.from_numpy(wide, dtype=dtype)
            self.dq, self.dk, self.dv = dev[:, :hq], dev[:, hq:hq + hkv], dev[:, hq + hkv:]
        else:
            self.dq, self.dk, self.dv = (DeviceArray.from_numpy(np.ascontiguousarray(a), dtype=dtype)
                                         for a in (self.q, self.k, self.v))
        self.pos = rng.integers(0, rows, T)
        self.table = mk.rotary_table(rows, rot)
        self.cs = self.table.to_numpy()[self.pos]
        wdtype = wdtype or dtype
        self.qw = kv_oracle.round_to((1 + 0.2 * rng.standard_normal(d)).astype(np.float32), wdtype) if norm else None
        self.kw = kv_oracle.round_to((1 + 0.2 * rng.standard_normal(d)).astype(np.float32), wdtype) if norm else None
        self.w = dict(q_weight=DeviceArray.from_numpy(self.qw, dtype=wdtype),
                      k_weight=DeviceArray.from_numpy(self.kw, dtype=wdtype)) if norm else {}

    def want(self, interleaved, eps=1e-6):
        return (plain_rope(self.q, self.qw, self.cs, self.rot, interleaved, eps),
                plain_rope(self.k, self.kw, self.cs, self.rot, interleaved, eps))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("d,rot", [(128, 128), (128, 64), (64, 64), (64, 2), (80, 80), (80, 40), (96, 96), (256, 256),
                                   (256, 64), (120, 24), (10, 6), (7, 4), (512, 128), (32, 16)])
def test_qk_norm_rope_head_sizes(gpu, d, rot, dtype, interleaved):
    for norm in (False, True):
        c = Rope(d + rot, dtype, 9, 5, 2, d, rot, norm)
        q, k = mk.qk_norm_rope(c.dq, c.dk, c.pos.astype(np.int64), c.table, interleaved=interleaved, **c.w)
        for g, w in zip((q, k), c.want(interleaved)):
            close(g.to_numpy(), w, dtype)
    assert _lib.get_status(0, clear=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T,hq,hkv", [(1, 1, 1), (1, 32, 8), (2, 28, 4), (700, 32, 8), (33, 64, 8), (1500, 3, 1)])
@pytest.mark.parametrize("fused", [False, True])
def test_qk_norm_rope_shapes(gpu, T, hq, hkv, fused):
    c = Rope(T, "bfloat16", T, hq, hkv, 128, 128, True, "float32", fused)
    q, k = mk.qk_norm_rope(c.dq, c.dk, c.pos.astype(np.int32), c.table, eps=1e-5, **c.w)
    for g, w in zip((q, k), c.want(False, 1e-5)):
        close(g.to_numpy(), w, "bfloat16")


@pytest.mark.gpu
@pytest.mark.parametrize("d,rot", [(128, 128), (10, 10)])
def test_qk_norm_rope_in_place_one_weight_and_padding(gpu, d, rot):
    c = Rope(5, "bfloat16", 40, 6, 2, d, rot, True, fused=False)
    pos = c.pos.copy()
    pos[3], pos[17], pos[39] = -1, 5000, -9  # padding, past the table, padding
    want_q, _ = c.want(True)
    want_k = plain_rope(c.k, None, c.cs, rot, True, 0.0)
    want_q[[3, 17, 39]], want_k[[3, 17, 39]] = c.q[[3, 17, 39]], c.k[[3, 17, 39]]
    s = Stream()
    mk.synchronize()
    mk.qk_norm_rope(c.dq, c.dk, DeviceArray.from_numpy(pos.astype(np.int32)), c.table, q_weight=c.w["q_weight"],
                    interleaved=True, q_out=c.dq, k_out=c.dk, stream=s)
    s.synchronize()
    close(c.dq.to_numpy(), want_q, "bfloat16")
    close(c.dk.to_numpy(), want_k, "bfloat16")
    assert _lib.get_status(0, clear=True) == _lib.STATUS_INDEX_OOB


@pytest.mark.gpu
def test_qk_norm_rope_zero_rows_and_unrotated_infinities(gpu):
    """A row of zeros stays zero; elements past the rotated part pass as they are."""
    c = Rope(6, "float16", 3, 2, 1, 128, 64, True, fused=False)
    x = np.zeros((3, 2, 128), np.float32)
    q, _ = mk.qk_norm_rope(DeviceArray.from_numpy(x, dtype="float16"), c.dk, c.pos.astype(np.int32), c.table, **c.w)
    assert not q.to_numpy().any()
    x[1, 0, 70:75] = [np.inf, -np.inf, 3.0, np.nan, 1.0]
    q, _ = mk.qk_norm_rope(DeviceArray.from_numpy(x, dtype="float16"), c.dk, c.pos.astype(np.int32), c.table)
    np.testing.assert_array_equal(q.to_numpy(), x)


# ---- with the append ------------------------------------------------------------------


def cache_shapes(layout, blocks, bs, hkv, d, dtype):
    x = 16 // dtypes.itemsize(dtype)
    return {"paged": ((blocks, hkv, d // x, bs, x), (blocks, hkv, d, bs)), "flash": ((blocks, bs, hkv, d),) * 2,
            "pool": ((blocks * bs, hkv, d),) * 2}[layout]


def place(layout, kc, vc, slots, k, v, bs):
    for t, s in enumerate(slots):
        if s < 0 or s >= kc.shape[0] * (1 if layout == "pool" else bs):
            continue
        if layout == "paged":
            kc[s // bs, :, :, s % bs, :] = k[t].reshape(k.shape[1], -1, kc.shape[-1])
            vc[s // bs, :, :, s % bs] = v[t]
        elif layout == "flash":
            kc[s // bs, s % bs], vc[s // bs, s % bs] = k[t], v[t]
        else:
            kc[s], vc[s] = k[t], v[t]


@pytest.mark.gpu
@pytest.mark.parametrize("layout,bs", [("paged", 8), ("paged", 16), ("paged", 32), ("flash", 16), ("flash", 5),
                                       ("pool", 1)])
@pytest.mark.parametrize("dtype,cache,d,rot,T", [
    ("bfloat16", "bfloat16", 128, 128, 50), ("bfloat16", "bfloat16", 128, 64, 1), ("float16", "float16", 64, 64, 1333),
    ("float16", "float16", 80, 40, 20), ("float32", "float32", 96, 96, 1100), ("float32", "float16", 128, 128, 30),
    ("float32", "bfloat16", 64, 64, 30), ("bfloat16", "bfloat16", 256, 256, 1025), ("float16", "float16", 120, 24, 9)])
def test_append(gpu, layout, bs, dtype, cache, d, rot, T):
    if layout != "paged" and cache != dtype:
        pytest.skip("token-major caches take their own dtype (refused, see below)")
    c = Rope(T + d, dtype, T, 4, 3, d, rot, T % 2 == 0)
    rng = np.random.default_rng(T)
    blocks = -(-T // bs) * 2 + 2
    # runs of consecutive slots and scattered ones, some padding, one past the cache
    slots = np.concatenate([np.arange(T // 2) + 3, rng.permutation(np.arange(T // 2 + 3, blocks * bs))[:T - T // 2]])
    flagged = 0
    if T > 8:
        slots[4] = -1
        slots[7] = blocks * bs + 5
        flagged = _lib.STATUS_SLOT_OOB
    ks, vs = cache_shapes(layout, blocks, bs, 3, d, cache)
    kc0 = kv_oracle.round_to(rng.standard_normal(ks).astype(np.float32), cache)
    vc0 = kv_oracle.round_to(rng.standard_normal(vs).astype(np.float32), cache)
    kc, vc = DeviceArray.from_numpy(kc0, dtype=cache), DeviceArray.from_numpy(vc0, dtype=cache)
    for idt in (np.int32, np.int64):
        q, _, _ = mk.qk_norm_rope_append(c.dq, c.dk, c.dv, c.pos.astype(idt), c.table, kc, vc, slots.astype(idt),
                                         interleaved=d == 64, **c.w)
        want_q, want_k = c.want(d == 64)
        close(q.to_numpy(), want_q, dtype)
        kw, vw = kc0.astype(np.float64), vc0.astype(np.float64)
        place(layout, kw, vw, slots, want_k, kv_oracle.round_to(c.v, cache), bs)
        close(kc.to_numpy(), kw, cache)
        np.testing.assert_array_equal(vc.to_numpy(), vw.astype(np.float32))
        assert _lib.get_status(0, clear=True) == flagged


# Many tokens: from 7 * 148 = 1036 of them with 128 * 148 = 18944 groups (a group: the rows of one tensor that a warp
# holds at a time, 4 heads of 64, 2 of 80 to 128, 1 of 256) a warp takes all of a token's rows, through its lanes' copy rings.
MANY = [(1100, 128, 128), (1100, 128, 64), (1900, 64, 64), (1100, 80, 40), (1040, 256, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("T,d,rot", MANY)
def test_qk_norm_rope_many_tokens(gpu, T, d, rot, dtype, interleaved):
    """Slices of a fused projection with norms, and in place without a norm of k, with skipped tokens."""
    c = Rope(T + rot, dtype, T, 32, 8, d, rot, True, "float32" if rot == 64 else None)
    q, k = mk.qk_norm_rope(c.dq, c.dk, c.pos.astype(np.int32), c.table, interleaved=interleaved, **c.w)
    want_q, want_k = c.want(interleaved)
    close(q.to_numpy(), want_q, dtype)
    close(k.to_numpy(), want_k, dtype)
    pos = c.pos.copy()
    skipped = [0, 500, T - 1]
    pos[skipped] = -1, 5000, -7
    want_k = plain_rope(c.k, None, c.cs, rot, interleaved, 0.0)
    want_q[skipped], want_k[skipped] = c.q[skipped], c.k[skipped]
    mk.qk_norm_rope(c.dq, c.dk, pos.astype(np.int64), c.table, q_weight=c.w["q_weight"], interleaved=interleaved,
                    q_out=c.dq, k_out=c.dk)
    close(c.dq.to_numpy(), want_q, dtype)
    close(c.dk.to_numpy(), want_k, dtype)
    assert _lib.get_status(0, clear=True) == _lib.STATUS_INDEX_OOB


@pytest.mark.gpu
@pytest.mark.parametrize("layout,bs", [("paged", 16), ("paged", 32), ("flash", 16), ("pool", 1)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("T,d,rot", MANY)
def test_append_many_tokens(gpu, T, d, rot, dtype, layout, bs):
    c = Rope(T + d, dtype, T, 32, 8, d, rot, rot != 64, fused=bs != 1)
    rng = np.random.default_rng(T + bs)
    blocks = -(-T // bs) * 2 + 2
    slots = np.concatenate([np.arange(T // 2) + 3, rng.permutation(np.arange(T // 2 + 3, blocks * bs))[:T - T // 2]])
    slots[4], slots[7] = -1, blocks * bs + 5
    ks, vs = cache_shapes(layout, blocks, bs, 8, d, dtype)
    kc0 = kv_oracle.round_to(rng.standard_normal(ks).astype(np.float32), dtype)
    vc0 = kv_oracle.round_to(rng.standard_normal(vs).astype(np.float32), dtype)
    kc, vc = DeviceArray.from_numpy(kc0, dtype=dtype), DeviceArray.from_numpy(vc0, dtype=dtype)
    interleaved = bs == 32 or d == 80
    q, _, _ = mk.qk_norm_rope_append(c.dq, c.dk, c.dv, c.pos.astype(np.int32), c.table, kc, vc, slots.astype(np.int64),
                                     interleaved=interleaved, **c.w)
    want_q, want_k = c.want(interleaved)
    close(q.to_numpy(), want_q, dtype)
    kw, vw = kc0.astype(np.float64), vc0.astype(np.float64)
    place(layout, kw, vw, slots, want_k, c.v, bs)
    close(kc.to_numpy(), kw, dtype)
    np.testing.assert_array_equal(vc.to_numpy(), vw.astype(np.float32))
    assert _lib.get_status(0, clear=True) == _lib.STATUS_SLOT_OOB


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 1100])
def test_append_to_a_page_past_32_bits(gpu, T):
    """One block of 2^25 + 16 tokens: a head's page of 64 dims has more than 2^31 elements."""
    import torch

    bs, d = (1 << 25) + 16, 64
    c = Rope(T, "float16", T, 2, 1, d, d, False, fused=False)
    kc = torch.zeros((1, 1, d // 8, bs, 8), dtype=torch.float16, device="cuda")
    vc = torch.zeros((1, 1, d, bs), dtype=torch.float16, device="cuda")
    slots = np.arange(bs - T, bs)
    slots[:2] = 0, 1 << 24
    torch.cuda.synchronize()
    mk.qk_norm_rope_append(c.dq, c.dk, c.dv, c.pos.astype(np.int32), c.table, kc, vc, slots)
    mk.synchronize()
    at = torch.from_numpy(slots).cuda()
    got_k = kc[0, 0][:, at].permute(1, 0, 2).reshape(T, 1, d).float().cpu().numpy()
    close(got_k, c.want(False)[1], "float16")
    np.testing.assert_array_equal(vc[0, 0][:, at].t().reshape(T, 1, d).float().cpu().numpy(), c.v)
    kc[0, 0][:, at] = 0
    vc[0, 0][:, at] = 0
    assert not kc.view(torch.int32).any() and not vc.view(torch.int32).any()  # nothing anywhere else
    assert _lib.get_status(0, clear=True) == 0


@pytest.mark.gpu
def test_append_skipped_position_keeps_the_value(gpu):
    c = Rope(9, "bfloat16", 4, 4, 2, 128, 128, False)
    pos = np.array([5, -1, 7, 9], np.int32)
    ks, vs = cache_shapes("paged", 4, 16, 2, 128, "bfloat16")
    kc, vc = DeviceArray.zeros(ks, "bfloat16"), DeviceArray.zeros(vs, "bfloat16")
    mk.qk_norm_rope_append(c.dq, c.dk, c.dv, pos, c.table, kc, vc, np.array([0, 17, 33, 50], np.int64))
    assert not kc.to_numpy()[1].any()
    np.testing.assert_array_equal(vc.to_numpy()[1, :, :, 1], c.v[1])
    assert _lib.get_status(0, clear=True) == 0


# ---- refusals ---------------------------------------------------------------------------


def _fake(shape, dtype="float16", strides=None):
    if strides is None:
        acc, st = 1, []
        for s in reversed(shape):
            st.append(acc)
            acc *= s
        strides = tuple(reversed(st))
    t, keep = dlpack.make_dltensor(0x10000, shape, strides, dtype, 0)
    _fake.keep.append(keep)
    return ctypes.pointer(t)


_fake.keep = []


def _rope_rc(q=(3, 4, 64), k=(3, 2, 64), pos=(3,), posd="int32", cs=(10, 64), csd="float32", w=(64,), wd="float16",
             qo=None, ko=None, eps=1e-6, kd="float16", qst=None):
    return _lib.lib.kvc_qk_norm_rope(_fake(qo or q), _fake(ko or k), _fake(q, strides=qst), _fake(k, kd),
                                     _fake(pos, posd), _fake(cs, csd), _fake(w, wd), None, eps, 0, None)


@pytest.mark.parametrize("kw,text", [
    (dict(k=(2, 2, 64)), "q must have shape"), (dict(kd="float32"), "must share"), (dict(pos=(2,)), "positions must be"),
    (dict(posd="uint32"), "positions must be int32 or int64"), (dict(cs=(10, 65)), "even rotary_dim"),
    (dict(cs=(10, 66)), "even rotary_dim"), (dict(csd="float16"), "cos_sin must be float32"),
    (dict(w=(32,)), "head_size entries"), (dict(wd="bfloat16"), "float32 or of q's dtype"),
    (dict(qo=(3, 4, 32)), "q_out must have"), (dict(ko=(3, 4, 64)), "k_out must have"), (dict(eps=-1.0), "eps must be"),
    (dict(eps=float("nan")), "eps must be"), (dict(qst=(256, 64, 2)), "must be contiguous"),
    (dict(q=(3, 4, 514), k=(3, 2, 514), cs=(10, 64), w=(514,)), "between 1 and 512")])
def test_rope_refusals(kw, text):
    assert _rope_rc(**kw) == 1
    assert text in _lib.last_error()


def test_append_refusals():
    def rc(kc=(5, 2, 8, 16, 8), vc=(5, 2, 64, 16), slots=(3,), sd="int64", v=(3, 2, 64), cd="float16", qd="float16"):
        return _lib.lib.kvc_qk_norm_rope_append(
            _fake((3, 4, 64), qd), _fake(kc, cd), _fake(vc, cd), _fake((3, 4, 64), qd), _fake((3, 2, 64), qd), _fake(v, qd),
            _fake((3,), "int32"), _fake((10, 64), "float32"), None, None, 1e-6, 0, _fake(slots, sd), None)

    for kw, text in ((dict(slots=(2,)), "slot_mapping must have shape"), (dict(sd="uint32"), "int32 or int64"),
                     (dict(v=(3, 4, 64)), "key and value must both"), (dict(kc=(5, 3, 8, 16, 8)), "KV-head count"),
                     (dict(cd="bfloat16"), "Unsupported dtype combination"),
                     (dict(kc=(5, 16, 2, 64), vc=(5, 16, 2, 64), qd="float32"), "dtypes to match")):
        assert rc(**kw) == 1
        assert text in _lib.last_error()


def test_step_tables_refusals():
    def rc(bt=(2, 4), kl=(2,), qi=(3,), po=(9,), sm=(9,), us=(1,), pl=(2,), nl=(2,), smd="int64", fd="int32", bs=16):
        return _lib.lib.kvc_step_tables(_fake(bt, "int32"), _fake(kl, "int32"), _fake(qi, "int32"), _fake(po, "int32"),
                                        _fake(sm, smd), _fake(us, "int32"), _fake(pl, "int32"), _fake(nl, "int32"),
                                        _fake((7,), fd), bs, None)

    for kw, text in ((dict(bt=(2,)), "block_tables must be 2D"), (dict(nl=(3,)), "num_seqs rows"),
                     (dict(qi=(2,)), "num_seqs + 1"), (dict(sm=(8,)), "same length"), (dict(bs=0), "block_size must be"),
                     (dict(smd="uint32"), "slot_mapping must be"), (dict(fd="int64"), "must be int32"),
                     (dict(kl=(2, 1)), "contiguous 1-D")):
        assert rc(**kw) == 1
        assert text in _lib.last_error()
    with pytest.raises(ValueError, match="num_tokens is needed"):
        mk.build_step_tables(None, None, object(), None, 16)


# what is laid out where: each array 64 KB from the next, as far as `at` does not say otherwise
_TABLE_ARGS = dict(bt=((3, 4), "int32"), kl=((3,), "int32"), qi=((4,), "int32"), po=((9,), "int32"), sm=((9,), "int64"),
                   us=((1,), "int32"), pl=((3,), "int32"), nl=((3,), "int32"), fb=((7,), "int32"))


@pytest.mark.parametrize("at", [
    dict(kl=("pl", 4)), dict(kl=("pl", -8)), dict(kl=("nl", 8)), dict(kl=("fb", 24)), dict(kl=("fb", 0)), dict(qi=("pl", 0)),
    dict(qi=("nl", 0)), dict(po=("pl", 8)), dict(sm=("nl", -68)), dict(us=("pl", 8)), dict(us=("fb", 0)), dict(po=("sm", 68)),
    dict(kl=("qi", 0)), dict(us=("kl", 4)), dict(bt=("fb", 24)), dict(fb=("bt", -24)), dict(kl=("bt", 44)), dict(pl=("bt", 0)),
    dict(kl=("pl", 0), nl=("pl", 4)), dict(kl=("nl", 0), po=("nl", 8))])
def test_step_tables_refuse_shared_memory(at):
    """Every CTA reads all lengths while others write: what is written must lie apart (kv_lens exactly on the lengths
    is allowed, and has a test of its own on a device)."""
    ptr = {n: 0x100000 + 0x10000 * i for i, n in enumerate(_TABLE_ARGS)}
    for n, (to, off) in at.items():
        ptr[n] = ptr[to] + off
    tensors = {}
    for n, (shape, dtype) in _TABLE_ARGS.items():
        strides = (4, 1) if len(shape) == 2 else (1,)
        t, keep = dlpack.make_dltensor(ptr[n], shape, strides, dtype, 0)
        tensors[n] = (ctypes.pointer(t), keep)
    rc = _lib.lib.kvc_step_tables(*(tensors[n][0] for n in ("bt", "kl", "qi", "po", "sm", "us", "pl", "nl", "fb")), 16, None)
    assert rc == 1 and "must not share memory" in _lib.last_error()


@pytest.mark.gpu
def test_step_tables_between_the_rows_of_a_wide_table(gpu):
    """Block tables that are a slice of wider rows, whose other columns hold the other arrays of the call."""
    import torch

    wide = torch.full((4, 64), -1, dtype=torch.int32, device="cuda")
    wide[0, 0], wide[1, 0] = 3, 9
    prefix, new = wide[1, 16:20], wide[2, 16:20]
    prefix.copy_(torch.tensor([5, 16, 0, 0]))
    new.copy_(torch.tensor([20, 1, 0, 17]))
    torch.cuda.synchronize()
    out = mk.build_step_tables(wide[:, :8], prefix, new, torch.tensor([10, 11, 12, 13], dtype=torch.int32, device="cuda"), 16,
                               38, kv_lens=wide[0, 24:28], qo_indptr=wide[3, 32:37])
    mk.synchronize()
    assert out.kv_lens.tolist() == [25, 17, 0, 17] and out.qo_indptr.tolist() == [0, 20, 21, 21, 38]
    assert wide[:, :3].tolist() == [[3, 10, -1], [9, 11, -1], [-1, -1, -1], [12, 13, -1]]
    assert prefix.tolist() == [5, 16, 0, 0] and new.tolist() == [20, 1, 0, 17]
    assert _lib.get_status(0, clear=True) == 0


def test_rotary_table_refusals():
    f = (ctypes.c_double * 32)(*([1.0] * 32))
    for t, text in (((_fake((4, 65), "float32")), "even rotary_dim"), (_fake((4, 258), "float32"), "even rotary_dim"),
                    (_fake((4, 64)), "must be float32")):
        assert _lib.lib.kvc_rotary_table(t, f, 1.0, None) == 1 and text in _lib.last_error()
    f[3] = math.inf
    assert _lib.lib.kvc_rotary_table(_fake((4, 64), "float32"), f, 1.0, None) == 1 and "finite" in _lib.last_error()
    with pytest.raises(ValueError):
        mk.rotary_table(0, 64)


# ---- the two ways into the library ----------------------------------------------


def _step_calls():
    """The five calls with preallocated outputs, on small inputs: (name, call) pairs; a call returns its outputs."""
    rng = np.random.default_rng(7)
    T, H, KH, D, bs, nb = 3, 4, 2, 64, 16, 8
    half = lambda *s: DeviceArray.from_numpy(rng.standard_normal(s).astype(np.float16))  # noqa: E731
    i32 = lambda a: DeviceArray.from_numpy(np.asarray(a, np.int32))  # noqa: E731
    q, k, v, w = half(T, H, D), half(T, KH, D), half(T, KH, D), half(D)
    kc, vc = half(nb, KH, D // 8, bs, 8), half(nb, KH, D, bs)
    rope = mk.rotary_table(40, D)
    pos, slots = i32([4, 17, 30]), DeviceArray.from_numpy(np.asarray([4, 33, 62], np.int64))
    tables, lens, ind = i32([[0, -1], [1, 2], [4, 3]]), i32([5, 18, 31]), i32([0, 1, 2, 3])
    like = lambda a: DeviceArray.zeros(a.shape, a.dtype)  # noqa: E731

    def tabs():
        t = i32(np.full((2, 4), -1))
        outs = [i32(np.zeros(n)) for n in (2, 3, 5)] + [DeviceArray.from_numpy(np.zeros(5, np.int64)), i32([0])]
        r = mk.build_step_tables(t, i32([0, 0]), i32([2, 3]), i32([5, 6, 7]), 4, kv_lens=outs[0], qo_indptr=outs[1],
                                 positions=outs[2], slot_mapping=outs[3], blocks_used=outs[4])
        return list(r)

    def append():
        kk, vv = like(kc), like(vc)
        return list(mk.qk_norm_rope_append(q, k, v, pos, rope, kk, vv, slots, q_weight=w, k_weight=w, q_out=like(q)))

    return [
        ("tables", tabs),
        ("rope", lambda: list(mk.qk_norm_rope(q, k, pos, rope, q_weight=w, k_weight=w, q_out=like(q), k_out=like(k)))),
        ("append", append),
        ("decode", lambda: [mk.paged_attention_window(q, kc, vc, tables, lens, KH, 0.125, bs, 32, 9, 2, out=like(q))]),
        ("extend", lambda: [mk.paged_prefill_window(q, kc, vc, tables, ind, lens, KH, 0.125, bs, 9, 2, max_q_len=1,
                                                    out=like(q))]),
    ]


@pytest.mark.gpu
def test_direct_calls_are_the_general_ones(gpu, monkeypatch):
    """With preallocated outputs a call goes to the library in one C call, where that module is built: the same bits."""
    direct = [[o.to_numpy(raw=True) for o in call()] for _, call in _step_calls()]
    monkeypatch.setattr(mk, "_calls", None)
    for (name, call), first in zip(_step_calls(), direct):
        for a, b in zip(call(), first):
            np.testing.assert_array_equal(a.to_numpy(raw=True), b, err_msg=name)
    assert _lib.get_status(0, clear=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("direct", [True, False])
def test_refusals_are_the_same_either_way(gpu, monkeypatch, direct):
    if not direct:
        monkeypatch.setattr(mk, "_calls", None)
    q = DeviceArray.zeros((2, 4, 64), "float16")
    kc, vc = DeviceArray.zeros((3, 2, 8, 16, 8), "float16"), DeviceArray.zeros((3, 2, 64, 16), "float16")
    t, n = DeviceArray.zeros((2, 1), "int32"), DeviceArray.zeros((2,), "int32")
    with pytest.raises(ValueError, match="window_size must be positive"):
        mk.paged_attention_window(q, kc, vc, t, n, 2, 0.125, 16, 16, 0, out=DeviceArray.zeros(q.shape, "float16"))
    with pytest.raises(ValueError, match="out"):
        mk.paged_attention_window(q, kc, vc, t, n, 2, 0.125, 16, 16, 4, out=DeviceArray.zeros((2, 4, 32), "float16"))


def test_direct_calls_are_built_for_this_interpreter():
    """Under the interpreter's own tag: another one does not load them (and calls through ctypes instead)."""
    import sysconfig

    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        pytest.skip("built without the interpreter's headers")
    assert mk._calls is not None
    assert mk._calls.__file__.endswith("_calls" + sysconfig.get_config_var("EXT_SUFFIX"))
    assert not os.path.exists(os.path.join(os.path.dirname(mk.__file__), "_calls.so"))


# ---- what a producer's tensors may be -------------------------------------------


def _cpu_calls():
    """The five calls on CPU torch tensors of fitting shapes, as (name, arguments, keywords, tensors' names)."""
    import torch

    f = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    q, k = f(3, 4, 64), f(3, 2, 64)
    kc, vc = f(8, 2, 8, 16, 8), f(8, 2, 64, 16)
    cs = torch.zeros(40, 64)
    slots = torch.zeros(3, dtype=torch.int64)
    return [
        ("paged_attention_window", [q, kc, vc, i(3, 2), i(3), 2, 0.125, 16, 32, 9, 2], dict(out=f(3, 4, 64))),
        ("paged_prefill_window", [q, kc, vc, i(3, 2), i(4), i(3), 2, 0.125, 16, 9, 2], dict(max_q_len=1, out=f(3, 4, 64))),
        ("build_step_tables", [i(3, 2), i(3), i(3), i(7), 16], dict(kv_lens=i(3), qo_indptr=i(4), positions=i(3),
                                                                  slot_mapping=slots, blocks_used=i(1))),
        ("qk_norm_rope", [q, k, i(3), cs], dict(q_weight=f(64), k_weight=f(64), q_out=f(3, 4, 64), k_out=f(3, 2, 64))),
        ("qk_norm_rope_append", [q, k, f(3, 2, 64), i(3), cs, kc, vc, slots], dict(q_weight=f(64), q_out=f(3, 4, 64))),
    ]


@pytest.mark.parametrize("direct", [True, False])
@pytest.mark.parametrize("stream", [None, 0])
@pytest.mark.parametrize("which", range(5))
def test_tensors_under_autograd_are_refused(monkeypatch, which, stream, direct):
    """As every other call does, through __dlpack__: a result would be cut off from the graph without a word."""
    if not direct:
        monkeypatch.setattr(mk, "_calls", None)
    name, args, kw = _cpu_calls()[which]
    for where in list(range(len(args))) + list(kw):
        name, args, kw = _cpu_calls()[which]
        t = args[where] if isinstance(where, int) else kw[where]
        if not (hasattr(t, "is_floating_point") and t.is_floating_point()):
            continue
        t.requires_grad_()
        with pytest.raises(BufferError, match="require gradient"):
            getattr(mk, name)(*args, **kw, stream=stream)
    name, args, kw = _cpu_calls()[which]  # (without one: what is wrong with these is that they are on the host)
    with pytest.raises(ValueError, match="CUDA device"):
        getattr(mk, name)(*args, **kw, stream=stream)


@pytest.mark.parametrize("direct", [True, False])
def test_tensors_that_are_not_strided_are_refused(monkeypatch, direct):
    import torch

    if not direct:
        monkeypatch.setattr(mk, "_calls", None)
    name, args, kw = _cpu_calls()[3]
    args[3] = torch.eye(40, 64).to_sparse()
    with pytest.raises(BufferError, match="strided"):
        getattr(mk, name)(*args, **kw)


@pytest.mark.parametrize("direct", [True, False])
def test_whole_numbers_past_32_bits(monkeypatch, direct):
    """A window or sinks past 2^31 (no limit) mean what they say, and other numbers do not wrap to small ones."""
    if not direct:
        monkeypatch.setattr(mk, "_calls", None)

    def call(which, at, value, name=None):
        fn, args, kw = _cpu_calls()[which]
        if name is None:
            args[at] = value
        else:
            kw[name] = value
        with pytest.raises(ValueError) as e:
            getattr(mk, fn)(*args, **kw)
        return str(e.value)

    for big in (2**31, 2**32, 2**32 + 5, 2**63, 2**80):
        for which, at in ((0, 9), (0, 10), (1, 9), (1, 10)):  # windows and sinks: as far as the tensors, which are on the host
            assert "CUDA device" in call(which, at, big)
        assert "max_seq_len exceeds" in call(0, 8, big)
        assert "num_heads must be divisible" in call(0, 5, big) and "num_heads must be divisible" in call(1, 6, big)
        assert "match block_size" in call(0, 7, big) and "match block_size" in call(1, 8, big)
        assert "CUDA device" in call(1, None, big, "max_q_len")
        assert "window_size must be positive" in call(0, 9, -big) and "sink_size must be" in call(1, 10, -big)
        assert "block_size must be positive" in call(2, 4, -big)


@pytest.mark.parametrize("direct", [True, False])
def test_a_negative_bound_on_new_tokens_is_refused(monkeypatch, direct):
    """On both ways into the library: nothing would be written."""
    if not direct:
        monkeypatch.setattr(mk, "_calls", None)
    for out in (True, False):
        name, args, kw = _cpu_calls()[1]
        kw["max_q_len"] = -1
        if not out:
            kw["out"] = args[0]
        with pytest.raises(ValueError, match="max_q_len and window_size must be non-negative"):
            getattr(mk, name)(*args, **kw)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("direct", [True, False])
@pytest.mark.parametrize("which", range(5))
def test_tensors_without_memory_are_refused(monkeypatch, which, direct):
    """A tensor that has elements but no address (as tracing makes them) does not reach a kernel."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    if not direct:
        monkeypatch.setattr(mk, "_calls", None)
    with FakeTensorMode():
        name, args, kw = _cpu_calls()[which]
    with pytest.raises(ValueError, match="null data pointer"):
        getattr(mk, name)(*args, **kw, stream=0)


def test_descriptors_without_memory_are_refused():
    def null(shape, dtype="float16"):
        ptr = _fake(shape, dtype)
        ptr.contents.data = None
        return ptr

    assert _lib.lib.kvc_reshape_and_cache(_fake((3, 2, 64)), null((3, 2, 64)), _fake((5, 2, 8, 16, 8)),
                                          _fake((5, 2, 64, 16)), _fake((3,), "int64"), None) == 1
    assert "value: null data pointer" in _lib.last_error()
    assert _lib.lib.kvc_rotary_table(null((4, 64), "float32"), (ctypes.c_double * 32)(), 1.0, None) == 1
    assert "cos_sin: null data pointer" in _lib.last_error()


@pytest.mark.gpu
def test_an_error_is_returned_once(gpu):
    """A call that the CUDA runtime refused (here: a device that is not there) does not fail the calls after it."""
    for _, call in _step_calls():
        with pytest.raises(_lib.KVCacheError):
            _lib.get_status(99)
        call()
    assert _lib.get_status(0, clear=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("side", [False, True])
@pytest.mark.parametrize("direct", [True, False])
def test_torch_tensors_give_the_same_bits(gpu, monkeypatch, direct, side):
    """Through the exchange API, and from a stream other than the default one, which then is waited for."""
    import torch

    want = [[o.to_numpy(raw=True) for o in call()] for _, call in _step_calls()]
    if not direct:
        monkeypatch.setattr(mk, "_calls", None)

    def with_torch(fn):
        conv = lambda a: torch.from_dlpack(a) if isinstance(a, DeviceArray) else a  # noqa: E731
        return lambda *a, **k: fn(*map(conv, a), **{n: conv(v) for n, v in k.items()})

    for name in ("paged_attention_window", "paged_prefill_window", "build_step_tables", "qk_norm_rope", "qk_norm_rope_append"):
        monkeypatch.setattr(mk, name, with_torch(getattr(mk, name)))
    stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
    with torch.cuda.stream(stream):
        got = [call() for _, call in _step_calls()]
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            np.testing.assert_array_equal(a.cpu().numpy().view(b.dtype), b)
    assert _lib.get_status(0, clear=True) == 0


CAPTURED_STEPS = """
import sys
sys.path.insert(0, sys.argv[1])
import numpy as np
from sglang_mlx_b200 import _lib, metal_kernels as mk
from sglang_mlx_b200.device_array import DeviceArray, Graph, Stream

B, H, KH, D, bs, steps = 3, 8, 2, 128, 16, 9
rng = np.random.default_rng(1)
i32 = lambda a: DeviceArray.from_numpy(np.asarray(a, np.int32))
half = lambda *s: DeviceArray.from_numpy(rng.standard_normal(s).astype(np.float16))
q, k, v, w, rope = half(B, H, D), half(B, KH, D), half(B, KH, D), half(D), mk.rotary_table(4096, D)
k0, v0 = half(300, KH, D // 8, bs, 8).to_numpy(), half(300, KH, D, bs).to_numpy()
one, free, st = i32([1] * B), i32([299]), Stream()


class State:
    def __init__(self):
        self.kc, self.vc = DeviceArray.from_numpy(k0), DeviceArray.from_numpy(v0)
        self.lens, self.tables = i32([3, 2000, 1601]), i32(np.arange(3 * 126).reshape(3, 126) % 299)
        self.indptr, self.pos, self.used = i32([0] * (B + 1)), i32([0] * B), i32([0])
        self.slots = DeviceArray.from_numpy(np.zeros(B, np.int64))
        self.qr, self.out, self.out2 = (DeviceArray.zeros((B, H, D), "float16") for _ in range(3))

    def step(self):
        mk.build_step_tables(self.tables, self.lens, one, free, bs, kv_lens=self.lens, qo_indptr=self.indptr,
                             positions=self.pos, slot_mapping=self.slots, blocks_used=self.used, stream=st)
        mk.qk_norm_rope_append(q, k, v, self.pos, rope, self.kc, self.vc, self.slots, q_weight=w, k_weight=w,
                               q_out=self.qr, stream=st)
        mk.paged_attention_window(self.qr, self.kc, self.vc, self.tables, self.lens, KH, 0.09, bs, 2016, 900, 4, out=self.out,
                                  stream=st)
        mk.paged_prefill_window(self.qr, self.kc, self.vc, self.tables, self.indptr, self.lens, KH, 0.09, bs, 900, 4,
                                max_q_len=1, out=self.out2, stream=st)

    def seen(self):
        st.synchronize()
        return [a.to_numpy(raw=True) for a in (self.kc, self.vc, self.lens, self.pos, self.slots, self.out, self.out2)]


a, b = State(), State()
mk.synchronize()
graph = Graph.capture(st, a.step)  # (the first calls of the process)
for i in range(steps):
    graph.replay(st)
    b.step()
    for x, y in zip(a.seen(), b.seen()):
        np.testing.assert_array_equal(x, y)
assert a.lens.to_numpy().tolist() == [3 + steps, 2000 + steps, 1601 + steps] and a.pos.to_numpy()[1] == 2000 + steps - 1
assert _lib.get_status(0, clear=True) == 0
print("captured")
"""


@pytest.mark.gpu
def test_steps_captured_in_a_graph(gpu):
    """A decode step with its lengths on the device, captured before any of its calls has run, then replayed."""
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(mk.__file__))
    r = subprocess.run([sys.executable, "-c", CAPTURED_STEPS, root], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_the_stride_of_an_extent_of_one_is_nothing(gpu):
    """Producers leave any value there; no call reads it, or takes it for an alignment."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(3)
    half = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float16)  # noqa: E731

    def odd(t):
        return torch.as_strided(t, t.shape, [3 if n == 1 else st for n, st in zip(t.shape, t.stride())])

    q, k, v = half(1, 4, 64), half(1, 1, 64), half(1, 1, 64)
    kc, vc, tk, tv = half(1, 1, 8, 16, 8), half(1, 1, 64, 16), half(1, 16, 1, 64), half(1, 16, 1, 64)
    tables, lens = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.tensor([11], dtype=torch.int32, device="cuda")
    ind, pos = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([10], dtype=torch.int32, device="cuda")
    slot, cs = torch.tensor([10], device="cuda"), torch.randn((20, 64), generator=g, device="cuda")

    def run(f):
        a = (1, 0.125, 16, 16)
        kc1, vc1, tk1, tv1 = (f(t.clone()) for t in (kc, vc, tk, tv))
        mk.reshape_and_cache(f(k), f(v), kc1, vc1, f(slot))
        mk.qk_norm_rope_append(f(q), f(k), f(v), f(pos), cs, tk1, tv1, f(slot), q_out=f(q.clone()))
        outs = [kc1, vc1, tk1, tv1]
        outs += [mk.paged_attention_v1(f(q), kc1, vc1, f(tables), f(lens), *a)]
        outs += [mk.paged_attention_window(f(q), *c, f(tables), f(lens), *a, 5, 2) for c in ((kc1, vc1), (tk1, tv1))]
        outs += [mk.paged_prefill_window(f(q), *c, f(tables), ind, f(lens), 1, 0.125, 16, 5, 2) for c in ((kc1, vc1), (tk1, tv1))]
        mk.synchronize()
        return [o.cpu().numpy() if hasattr(o, "cpu") else o.to_numpy() for o in outs]

    for a, b in zip(run(odd), run(lambda t: t)):
        np.testing.assert_array_equal(a.reshape(-1), b.reshape(-1))
    assert _lib.get_status(0, clear=True) == 0
