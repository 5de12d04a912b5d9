"""Sliding-window attention with sinks (paged_attention_window,
paged_prefill_window) against the formula in float64: the query at position i
sees j <= i with j < sink_size or j > i - window_size."""

import ctypes

import numpy as np
import pytest

from helpers import assert_close, tolerance
from oracle import kv_oracle
from sglang_mlx_b200 import _lib, dlpack
from sglang_mlx_b200 import metal_kernels as mk
from sglang_mlx_b200.device_array import DeviceArray, Stream

NAN = float("nan")


def visible(i, window, sinks):
    j = np.arange(i + 1)
    return j[(j < sinks) | (j > i - window)]


def attend(q, K, V, i, window, sinks, scale, G, eps):
    """One query token [H, D] at position i over K, V [len, Hkv, D], float64."""
    j = visible(i, window, sinks)
    out = np.zeros(q.shape, np.float64)
    for h in range(q.shape[0]):
        s = K[j, h // G] @ q[h] * scale
        e = np.exp(s - s.max())
        out[h] = e @ V[j, h // G] / (e.sum() + eps)
    return out


class Case:
    """A ragged batch in a paged ("paged"), flash ("flash") or pool ("pool") cache."""

    def __init__(self, seed, dtype, lens, hq, hkv, d, bs, layout="paged", new=None, cache_dtype=None, spare=5):
        rng = np.random.default_rng(seed)
        self.lens, self.bs, self.layout, self.G = np.asarray(lens, np.int64), bs, layout, hq // hkv
        self.new = np.ones(len(lens), np.int64) if new is None else np.asarray(new, np.int64)
        self.dtype, self.cache_dtype = dtype, cache_dtype or dtype
        rows = int(self.new.sum())
        rnd = lambda shape, dt: kv_oracle.round_to(rng.standard_normal(shape).astype(np.float32), dt)  # noqa: E731
        self.q = rnd((rows, hq, d), dtype)
        need = -(-self.lens // bs)
        self.blocks = int(need.sum()) + spare
        perm = rng.permutation(self.blocks)
        width = int(max(1, need.max())) + 1
        self.tables = np.full((len(lens), width), -1, np.int64)
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = perm[at:at + n]
            at += n
        self.K = [rnd((int(n), hkv, d), self.cache_dtype) for n in self.lens]
        self.V = [rnd((int(n), hkv, d), self.cache_dtype) for n in self.lens]
        # what is not the cache of any sequence (the rest of last blocks, spare blocks) is NaN
        self.k_rows = np.full((self.blocks * bs, hkv, d), NAN, np.float32)
        self.v_rows = np.full((self.blocks * bs, hkv, d), NAN, np.float32)
        for b, n in enumerate(self.lens):
            t = np.arange(int(n))
            slot = self.tables[b, t // bs] * bs + t % bs
            self.k_rows[slot], self.v_rows[slot] = self.K[b], self.V[b]
        self.scale = d ** -0.5
        self.hkv, self.d = hkv, d
        self.indptr = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)

    def poison(self, window, sinks):
        """NaN into every cached token that no query sees, -1 into table entries of blocks without a seen token."""
        for b, n in enumerate(self.lens):
            seen = np.zeros(int(n), bool)
            for i in range(int(n - self.new[b]), int(n)):
                seen[visible(i, window, sinks)] = True
            t = np.nonzero(~seen)[0]
            slot = self.tables[b, t // self.bs] * self.bs + t % self.bs
            self.k_rows[slot] = self.v_rows[slot] = NAN
            for blk in range(-(-int(n) // self.bs)):
                if not seen[blk * self.bs:(blk + 1) * self.bs].any():
                    self.tables[b, blk] = -1

    def upload(self):
        hkv, d, bs, nb = self.hkv, self.d, self.bs, self.blocks
        kr, vr = self.k_rows.reshape(nb, bs, hkv, d), self.v_rows.reshape(nb, bs, hkv, d)
        if self.layout == "paged":
            x = 16 // (4 if self.cache_dtype == "float32" else 2)
            kr = kr.reshape(nb, bs, hkv, d // x, x).transpose(0, 2, 3, 1, 4)
            vr = vr.transpose(0, 2, 3, 1)
        elif self.layout == "pool":
            kr, vr = kr.reshape(nb * bs, hkv, d), vr.reshape(nb * bs, hkv, d)
        kc = DeviceArray.from_numpy(np.ascontiguousarray(kr), dtype=self.cache_dtype)
        vc = DeviceArray.from_numpy(np.ascontiguousarray(vr), dtype=self.cache_dtype)
        q = DeviceArray.from_numpy(self.q, dtype=self.dtype)
        return q, kc, vc, DeviceArray.from_numpy(self.tables.astype(np.int32)), DeviceArray.from_numpy(
            self.lens.astype(np.int32))

    @property
    def max_seq_len(self):
        return self.tables.shape[1] * self.bs

    def reference(self, window, sinks, eps):
        out = np.zeros(self.q.shape, np.float64)
        for b, n in enumerate(self.lens):
            K, V = self.K[b].astype(np.float64), self.V[b].astype(np.float64)
            for t in range(int(self.new[b])):
                i = int(n - self.new[b]) + t
                if i < 0 or n == 0:
                    continue
                r = int(self.indptr[b]) + t
                out[r] = attend(self.q[r].astype(np.float64), K, V, i, window, sinks, self.scale, self.G, eps)
        return out

    def decode(self, window, sinks, **kw):
        q, kc, vc, tables, lens = self.upload()
        return mk.paged_attention_window(q, kc, vc, tables, lens, self.hkv, self.scale, self.bs, self.max_seq_len,
                                         window, sinks, **kw).to_numpy()

    def extend(self, window, sinks, **kw):
        q, kc, vc, tables, lens = self.upload()
        return mk.paged_prefill_window(q, kc, vc, tables, self.indptr, lens, self.hkv, self.scale, self.bs, window,
                                       sinks, **kw).to_numpy()


LENS = [1, 2, 15, 16, 17, 33, 100, 257, 700, 1500]
WINDOWS = [(1, 0), (1, 1), (7, 0), (16, 4), (33, 17), (128, 64), (500, 3), (5000, 4)]


def check_decode(c, window, sinks, what=""):
    ref = c.reference(window, sinks, 1e-6)
    c.poison(window, sinks)
    got = c.decode(window, sinks)
    assert_close(got, ref, *tolerance(c.dtype), f"{what} window {window} sinks {sinks}")
    assert _lib.get_status(0, clear=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("layout,bs,d", [("paged", 8, 128), ("paged", 16, 128), ("paged", 32, 128), ("paged", 16, 64),
                                         ("paged", 32, 64), ("flash", 16, 128), ("flash", 32, 64), ("flash", 5, 128),
                                         ("flash", 24, 64), ("pool", 1, 128), ("pool", 1, 64)])
def test_decode_layouts(gpu, layout, bs, d, window, sinks):
    c = Case(11, "bfloat16", LENS, 8, 2, d, bs, layout)
    check_decode(c, window, sinks, f"{layout} {bs} {d}")


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 1), (16, 1), (28, 4), (8, 8), (40, 2)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_decode_head_groups(gpu, hq, hkv, dtype):
    check_decode(Case(12, dtype, [1, 40, 333], hq, hkv, 128, 16), 100, 4, f"{hq}/{hkv}")


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 80, 96, 112, 120, 128, 192, 256])
@pytest.mark.parametrize("dtype,cache", [("float32", "float32"), ("float32", "float16"), ("float32", "bfloat16"),
                                         ("float16", "float16"), ("bfloat16", "bfloat16")])
def test_decode_types_and_head_sizes(gpu, d, dtype, cache):
    check_decode(Case(13, dtype, [3, 70, 300], 6, 2, d, 8 if d == 120 else 16, cache_dtype=cache), 65, 9)


@pytest.mark.gpu
@pytest.mark.parametrize("n,window", [(1, 64), (1, 4096), (3, 1024), (40, 300)])
def test_decode_one_or_few_sequences(gpu, n, window):
    """Few (sequence, KV head) pairs: the seen tokens are split over a cluster."""
    rng = np.random.default_rng(n)
    check_decode(Case(14, "bfloat16", rng.integers(1, 9000, n), 8, 1, 128, 16), window, 4)
    check_decode(Case(15, "float32", rng.integers(1, 3000, n), 8, 1, 64, 32), window, 4)


@pytest.mark.gpu
def test_decode_zero_and_overlong_sequences(gpu):
    c = Case(16, "float16", [0, 5, 64, 0], 4, 2, 64, 16)
    ref = c.reference(8, 2, 1e-6)
    q, kc, vc, tables, lens = c.upload()
    out = mk.paged_attention_window(q, kc, vc, tables, lens, 2, c.scale, 16, 63, 8, 2).to_numpy()
    ref[2] = 0  # 64 tokens, past max_seq_len 63
    assert_close(out, ref, *tolerance("float16"))
    c32 = Case(16, "float32", [0, 5, 64, 0], 4, 2, 64, 16)
    q, kc, vc, tables, lens = c32.upload()
    out = mk.paged_attention_window(q, kc, vc, tables, lens, 2, c32.scale, 16, 63, 8, 2).to_numpy()
    ref = c32.reference(8, 2, 1e-6)
    ref[2] = 0
    assert_close(out, ref, *tolerance("float32"))


@pytest.mark.gpu
def test_decode_window_past_the_context_is_the_plain_decode(gpu):
    c = Case(17, "bfloat16", [7, 90, 600], 8, 2, 128, 16)
    q, kc, vc, tables, lens = c.upload()
    a = mk.paged_attention_window(q, kc, vc, tables, lens, 2, c.scale, 16, c.max_seq_len, 10000, 0).to_numpy()
    b = mk.paged_attention_v1(q, kc, vc, tables, lens, 2, c.scale, 16, c.max_seq_len).to_numpy()
    assert_close(a, b, 1e-6, 2.0 ** -7)  # two roundings of nearly the same value: one bfloat16 step


@pytest.mark.gpu
def test_decode_is_deterministic_and_strided(gpu):
    """The same bits every time; query and output rows may be slices of wider rows."""
    c = Case(18, "bfloat16", [9, 130, 1000], 8, 2, 128, 16)
    q, kc, vc, tables, lens = c.upload()
    wide = np.zeros((3, 12, 128), np.float32)
    wide[:, 2:10] = c.q
    qs = DeviceArray.from_numpy(wide, dtype="bfloat16")[:, 2:10]
    outw = DeviceArray.zeros((3, 11, 128), "bfloat16")
    args = (kc, vc, tables, lens, 2, c.scale, 16, c.max_seq_len, 100, 4)
    first = mk.paged_attention_window(q, *args).to_numpy(raw=True)
    for _ in range(3):
        np.testing.assert_array_equal(mk.paged_attention_window(q, *args).to_numpy(raw=True), first)
    s = Stream()
    mk.synchronize()
    mk.paged_attention_window(qs, *args, out=outw[:, 1:9], stream=s)
    s.synchronize()
    got = outw.to_numpy(raw=True)
    np.testing.assert_array_equal(got[:, 1:9], first)
    assert not got[:, :1].any() and not got[:, 9:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_decode_large_scores_and_infinite_unseen(gpu, sign):
    """Scores of +-1000 stay finite; infinities in unseen places do not matter."""
    c = Case(19, "float16", [300], 4, 1, 128, 16)
    c.q[:] = sign * 30.0
    c.K[0][:] = np.abs(c.K[0])
    c.k_rows[:] = np.inf
    t = np.arange(300)
    slot = c.tables[0, t // 16] * 16 + t % 16
    c.k_rows[slot] = c.K[0]
    check_decode(c, 50, 3)


@pytest.mark.gpu
def test_decode_bad_block_is_skipped_and_flagged(gpu):
    c = Case(20, "bfloat16", [200], 8, 2, 128, 16)
    q, kc, vc, _, lens = c.upload()
    t = c.tables.copy()
    t[0, 11] = c.blocks + 7  # tokens 176 .. 191, inside the window
    out = mk.paged_attention_window(q, kc, vc, DeviceArray.from_numpy(t.astype(np.int32)), lens, 2, c.scale, 16,
                                    c.max_seq_len, 40, 2).to_numpy()
    assert np.isfinite(out).all()
    assert _lib.get_status(0, clear=True) == _lib.STATUS_BLOCK_OOB


# ---- extend ---------------------------------------------------------------------


def check_extend(c, window, sinks, what=""):
    ref = c.reference(window, sinks, 0.0)
    c.poison(window, sinks)
    got = c.extend(window, sinks)
    assert_close(got, ref, *tolerance(c.dtype), f"{what} window {window} sinks {sinks}")
    assert _lib.get_status(0, clear=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("layout,bs,d", [("paged", 8, 128), ("paged", 16, 128), ("paged", 32, 128), ("paged", 16, 64),
                                         ("paged", 32, 64), ("flash", 16, 128), ("flash", 5, 64), ("pool", 1, 128)])
def test_extend_layouts(gpu, layout, bs, d, window, sinks):
    c = Case(31, "bfloat16", [1, 40, 130, 300, 555], 4, 2, d, bs, layout, new=[1, 40, 33, 1, 150])
    check_extend(c, window, sinks, f"{layout} {bs} {d}")


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,dtype", [(28, 4, "float16"), (8, 8, "float16"), (16, 1, "bfloat16"), (5, 1, "bfloat16")])
def test_extend_head_groups(gpu, hq, hkv, dtype):
    check_extend(Case(32, dtype, [77, 400], hq, hkv, 128, 16, new=[77, 90]), 100, 4)


@pytest.mark.gpu
def test_extend_many_sequences_and_a_long_prefix(gpu):
    rng = np.random.default_rng(33)
    new = rng.integers(0, 30, 60)
    lens = new + rng.integers(0, 200, 60)
    lens[7] = new[7] + 5000
    check_extend(Case(33, "bfloat16", lens, 4, 1, 64, 32, new=new), 64, 20)


@pytest.mark.gpu
@pytest.mark.parametrize("layout,bs,d", [("paged", 32, 128), ("paged", 16, 64), ("flash", 16, 64), ("pool", 1, 128)])
def test_extend_more_items_than_sms(gpu, layout, bs, d):
    """Each CTA takes several (128-row tile, sequence, KV head) items, of one tile and of more."""
    rng = np.random.default_rng(35)
    new = rng.integers(1, 60, 100)
    lens = new + rng.integers(0, 400, 100)
    check_extend(Case(35, "bfloat16", lens, 16, 4, d, bs, layout, new=new), 150, 4)


@pytest.mark.gpu
def test_extend_of_one_token(gpu):
    check_extend(Case(34, "float16", [5, 64, 700], 8, 2, 64, 16), 90, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("layout,bs,d", [("paged", 8, 128), ("paged", 16, 128), ("paged", 32, 128), ("paged", 16, 64),
                                         ("paged", 32, 64), ("flash", 16, 128), ("flash", 32, 64), ("flash", 5, 64),
                                         ("pool", 1, 128), ("pool", 1, 64)])
def test_extend_few_tokens(gpu, layout, bs, d, window, sinks):
    """At most one 16-row tile to an SM: tiles of several tokens, whole and ragged, split over a cluster."""
    c = Case(36, "bfloat16", [1, 40, 133, 300, 555, 2000], 6, 2, d, bs, layout, new=[1, 7, 33, 0, 20, 2])
    check_extend(c, window, sinks, f"{layout} {bs} {d}")


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [2, 8, 40])
def test_extend_unaligned_output_rows(gpu, seqs):
    """Output rows that start at 4 bytes past a 16-byte boundary, from few 16-row tiles to many."""
    rng = np.random.default_rng(37)
    new = rng.integers(20, 61, seqs)
    c = Case(37, "bfloat16", new + rng.integers(0, 300, seqs), 16, 4, 128, 16, new=new)
    ref = c.reference(70, 3, 0.0)
    q, kc, vc, tables, lens = c.upload()
    wide = DeviceArray.zeros((q.shape[0], 16, 136), "bfloat16")
    mk.paged_prefill_window(q, kc, vc, tables, c.indptr, lens, 4, c.scale, 16, 70, 3, out=wide[:, :, 2:130])
    got = wide.to_numpy()
    assert_close(got[:, :, 2:130], ref, *tolerance("bfloat16"))
    assert not got[:, :, :2].any() and not got[:, :, 130:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [2, 40])
@pytest.mark.parametrize("bs", [5, 16])
def test_extend_strided_token_rows(gpu, seqs, bs):
    """A token-major cache that is a slice of wider rows."""
    rng = np.random.default_rng(38)
    new = rng.integers(20, 61, seqs)
    c = Case(38, "float16", new + rng.integers(0, 300, seqs), 16, 4, 64, bs, "flash", new=new)
    ref = c.reference(70, 3, 0.0)
    q, _, _, tables, lens = c.upload()
    caches = []
    for rows in (c.k_rows, c.v_rows):
        wide = np.full((c.blocks, bs, 6, 64), NAN, np.float32)
        wide[:, :, 1:5] = rows.reshape(c.blocks, bs, 4, 64)
        caches.append(DeviceArray.from_numpy(wide, dtype="float16")[:, :, 1:5])
    got = mk.paged_prefill_window(q, caches[0], caches[1], tables, c.indptr, lens, 4, c.scale, bs, 70, 3).to_numpy()
    assert_close(got, ref, *tolerance("float16"))


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [2, 40])
@pytest.mark.parametrize("layout,bs,pad", [("paged", 16, 8), ("paged", 32, 8), ("paged", 8, 64), ("flash", 16, 8),
                                           ("flash", 5, 8), ("flash", 5, 256), ("flash", 16, 512)])
def test_extend_blocks_any_distance_apart(gpu, layout, bs, pad, seqs):
    """Elements between one block and the next: whole K chunks or token rows (which tensor maps can step over) or not."""
    import torch

    rng = np.random.default_rng(42)
    new = rng.integers(20, 61, seqs)
    c = Case(42, "float16", new + rng.integers(0, 300, seqs), 16, 4, 64, bs, layout, new=new)
    ref = c.reference(70, 3, 0.0)
    q, kc, vc, tables, lens = c.upload()
    spread = []
    for a in (kc, vc):
        a = torch.from_numpy(a.to_numpy())
        flat = torch.full((c.blocks, a[0].numel() + pad), NAN, dtype=torch.float16)
        flat[:, :a[0].numel()] = a.reshape(c.blocks, -1)
        spread.append(torch.as_strided(flat.cuda(), a.shape, (flat.shape[1],) + a.stride()[1:]))
    torch.cuda.synchronize()
    got = mk.paged_prefill_window(q, spread[0], spread[1], tables, c.indptr, lens, 4, c.scale, bs, 70, 3).to_numpy()
    assert_close(got, ref, *tolerance("float16"))
    assert _lib.get_status(0, clear=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [3, 40])
def test_extend_index_errors(gpu, seqs):
    """Lengths that the host cannot see: the status word names the error, the sequence's
    rows are 0, rows past the query are not written, and the other sequences are right."""
    rng = np.random.default_rng(39)
    new = rng.integers(20, 61, seqs)
    c = Case(39, "bfloat16", new + rng.integers(0, 300, seqs), 16, 4, 64, 16, new=new)
    ref = c.reference(70, 3, 0.0)
    q, kc, vc, tables, _ = c.upload()
    for bad in (int(new[1]) - 1, c.max_seq_len + 1):
        kl = c.lens.astype(np.int32)
        kl[1] = bad
        _lib.get_status(0, clear=True)
        got = mk.paged_prefill_window(q, kc, vc, tables, c.indptr, kl, 4, c.scale, 16, 70, 3).to_numpy()
        assert _lib.get_status(0, clear=True) == _lib.STATUS_INDEX_OOB
        want = ref.copy()
        want[c.indptr[1]:c.indptr[2]] = 0
        assert_close(got, want, *tolerance("bfloat16"))
    last = int(c.indptr[-2])  # the last sequence reaches past a query one row shorter than its tokens
    out = DeviceArray.zeros(q.shape, "bfloat16")
    mk.paged_prefill_window(q[:-1], kc, vc, tables, DeviceArray.from_numpy(c.indptr), c.lens.astype(np.int32), 4, c.scale,
                            16, 70, 3, max_q_len=int(new.max()), out=out[:-1])
    assert _lib.get_status(0, clear=True) == _lib.STATUS_INDEX_OOB
    got = out.to_numpy()
    assert_close(got[:last], ref[:last], *tolerance("bfloat16"))
    assert not got[last:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [3, 60])
@pytest.mark.parametrize("sinks", [4, 0])
@pytest.mark.parametrize("layout,bs,d", [("paged", 32, 128), ("paged", 32, 64), ("paged", 16, 128), ("paged", 8, 64),
                                         ("flash", 32, 64), ("flash", 16, 128), ("flash", 5, 128), ("pool", 1, 64)])
def test_extend_bad_blocks_are_skipped(gpu, layout, bs, d, seqs, sinks):
    """Blocks past the cache are flagged and their tokens left out, whatever a row's other blocks, the unseen
    places of those, or the sequences that ran before on the same SM hold."""
    rng = np.random.default_rng(40 + bs)
    new = rng.integers(20, 61, seqs)
    c = Case(40, "bfloat16", new + rng.integers(0, 400, seqs), 16, 4, d, bs, layout, new=new)
    window, flagged = 150, 0
    # every third sequence misses a fifth of its blocks, among them neither the first nor the last two tokens'
    lost = [np.zeros(int(n), bool) for n in c.lens]
    bad = c.tables.copy()
    for b in range(0, seqs, 3):
        n = int(c.lens[b])
        for blk in rng.permutation(np.arange(1, max(1, (n - 2) // bs)))[:max(1, n // bs // 5)]:
            bad[b, blk] = c.blocks + int(rng.integers(0, 1000))
            lost[b][blk * bs:(blk + 1) * bs] = True
    ref = np.zeros(c.q.shape, np.float64)
    for b, n in enumerate(c.lens):
        for t in range(int(new[b])):
            i, r = int(n - new[b]) + t, int(c.indptr[b]) + t
            j = visible(i, window, sinks)
            flagged |= _lib.STATUS_BLOCK_OOB if lost[b][j].any() else 0
            j = j[~lost[b][j]]
            for h in range(16 if len(j) else 0):
                s = c.K[b][j, h // 4].astype(np.float64) @ c.q[r, h].astype(np.float64) * c.scale
                e = np.exp(s - s.max())
                ref[r, h] = e @ c.V[b][j, h // 4].astype(np.float64) / e.sum()
    c.poison(window, sinks)
    c.tables = np.where(bad >= c.blocks, bad, c.tables)
    _lib.get_status(0, clear=True)
    for _ in range(3):  # (the order of the items over the SMs is not fixed)
        got = c.extend(window, sinks)
        assert_close(got, ref, *tolerance("bfloat16"))
        assert _lib.get_status(0, clear=True) == flagged


@pytest.mark.gpu
@pytest.mark.parametrize("value", [NAN, np.inf])
@pytest.mark.parametrize("dtype,d", [("float16", 128), ("bfloat16", 64), ("float32", 96)])
def test_decode_nan_that_is_seen_shows(gpu, dtype, d, value):
    """A key that is not finite makes the result of whoever sees it NaN, as the formula does, and of nobody else."""
    c = Case(44, dtype, [300, 300, 300, 40], 4, 2, d, 16)
    for b, j in ((0, 290), (1, 200), (3, 1)):  # in the window, in the gap, a sink
        c.k_rows[c.tables[b, j // 16] * 16 + j % 16] = value
        c.K[b][j] = value
    c.q = kv_oracle.round_to(np.abs(c.q) + 0.5, c.dtype)
    with np.errstate(invalid="ignore"):
        ref = c.reference(50, 2, 1e-6)
    assert np.isnan(ref[[0, 3]]).all() and np.isfinite(ref[[1, 2]]).all()
    got = c.decode(50, 2)
    assert np.isnan(got[[0, 3]]).all()
    assert_close(got[[1, 2]], ref[[1, 2]], *tolerance(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [2, 40])
@pytest.mark.parametrize("layout,bs", [("paged", 16), ("flash", 16), ("pool", 1)])
@pytest.mark.parametrize("value", [NAN, np.inf])
def test_extend_nan_that_is_seen_shows(gpu, layout, bs, seqs, value):
    rng = np.random.default_rng(45)
    new = rng.integers(20, 61, seqs)
    c = Case(45, "bfloat16", new + rng.integers(60, 300, seqs), 16, 4, 64, bs, layout, new=new)
    c.q = kv_oracle.round_to(np.abs(c.q) + 0.5, c.dtype)
    for b in range(0, seqs, 2):
        j = int(c.lens[b] - c.new[b] // 2)  # seen by the later half of the new tokens
        c.k_rows[c.tables[b, j // bs] * bs + j % bs] = value
        c.K[b][j] = value
    with np.errstate(invalid="ignore"):
        ref = c.reference(70, 3, 0.0)
    nan = np.isnan(ref)
    assert nan.any() and not nan.all()
    got = c.extend(70, 3)
    np.testing.assert_array_equal(np.isnan(got), nan)
    assert_close(got[~nan], ref[~nan], *tolerance("bfloat16"))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["decode", "decode fp32", "decode pool", "few", "many"])
def test_output_is_the_next_query(gpu, kind):
    """A kernel may start before the one ahead of it on the stream has ended, but reads nothing that this one writes
    before it has: an attention output as the next call's query."""
    dtype = "float32" if "fp32" in kind else "bfloat16"
    new = None if kind.startswith("decode") else [9, 4] if kind == "few" else [700, 500]
    layout, bs = ("pool", 1) if "pool" in kind else ("paged", 16)
    a = Case(46, dtype, [9000, 7000], 8, 2, 128, bs, layout, new=new)
    q, kc, vc, tables, lens = a.upload()
    ind = DeviceArray.from_numpy(a.indptr)
    window = 6000 if kind.startswith("decode") else 900

    def call(query, lens, out):
        if kind.startswith("decode"):
            return mk.paged_attention_window(query, kc, vc, tables, lens, 2, a.scale, bs, a.max_seq_len, window, 3, out=out)
        return mk.paged_prefill_window(query, kc, vc, tables, ind, lens, 2, a.scale, bs, window, 3,
                                       max_q_len=max(new), out=out)

    outs = [DeviceArray.zeros(q.shape, dtype) for _ in range(6)]
    apart = [DeviceArray.zeros(q.shape, dtype) for _ in range(6)]
    for _ in range(3):
        for i in range(6):  # (one after another)
            call(apart[i - 1] if i else q, lens, apart[i])
            mk.synchronize()
        for o in outs:
            o.fill_zero()
        mk.synchronize()
        for i in range(6):
            call(outs[i - 1] if i else q, lens, outs[i])
        for i in range(6):
            np.testing.assert_array_equal(outs[i].to_numpy(raw=True), apart[i].to_numpy(raw=True), err_msg=f"{kind} {i}")


@pytest.mark.gpu
@pytest.mark.parametrize("factor", [2, 3, 8])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("layout,bs,d", [("paged", 16, 64), ("paged", 32, 128), ("flash", 16, 64), ("pool", 1, 128)])
def test_extend_with_few_large_weights(gpu, layout, bs, d, dtype, factor):
    """Scores of standard deviation `factor`: a few keys have most of a row's weight, and where their values nearly
    cancel the weights' own rounding shows.  The tolerance is that of every other case."""
    rng = np.random.default_rng(47)
    new = rng.integers(30, 91, 40)
    c = Case(47, dtype, new + rng.integers(0, 300, 40), 16, 4, d, bs, layout, new=new)
    c.q = kv_oracle.round_to(c.q * factor, dtype)
    check_extend(c, 130, 3, f"{layout} {dtype} x{factor}")


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [2, 40])
def test_extend_bits_repeat(gpu, seqs):
    """The same call gives the same bits, on any stream; max_q_len may be larger than needed."""
    rng = np.random.default_rng(41)
    new = rng.integers(20, 61, seqs)
    c = Case(41, "bfloat16", new + rng.integers(0, 900, seqs), 16, 4, 128, 32, new=new)
    ref = c.reference(200, 3, 0.0)
    q, kc, vc, tables, lens = c.upload()
    args = (q, kc, vc, tables, DeviceArray.from_numpy(c.indptr), lens, 4, c.scale, 32, 200, 3)
    for longest in (int(new.max()), q.shape[0]):
        first = mk.paged_prefill_window(*args, max_q_len=longest)
        assert_close(first.to_numpy(), ref, *tolerance("bfloat16"))
        for _ in range(3):
            s = Stream()
            out = DeviceArray.zeros(q.shape, "bfloat16")
            mk.synchronize()
            mk.paged_prefill_window(*args, max_q_len=longest, out=out, stream=s)
            s.synchronize()
            np.testing.assert_array_equal(out.to_numpy(raw=True), first.to_numpy(raw=True))


@pytest.mark.gpu
def test_window_serving_example(gpu):
    """The example's chunked prompts and decode steps, blocks behind the window reused.  Tolerance: values of at
    most about 4.5, one fp16 rounding of the output (2^-11 relative) and of P (2^-11 each), of the rotated q and
    the cached k where the fp32 result rounds differently (one step, rare): under 4 x 4.5 x 2^-11 = 8.8e-3."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(__file__), "..", "examples", "window_serving.py")
    spec = importlib.util.spec_from_file_location("window_serving", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    lines = []
    assert example.main(steps=24, requests=5, log=lines.append) < 8.8e-3
    assert len(lines) == 24 and _lib.get_status(0, clear=True) == 0


# ---- refusals -------------------------------------------------------------------


def _fake(shape, dtype="float16"):
    acc, st = 1, []
    for s in reversed(shape):
        st.append(acc)
        acc *= s
    t, keep = dlpack.make_dltensor(0x10000, shape, tuple(reversed(st)), dtype, 0)
    _fake.keep.append(keep)
    return ctypes.pointer(t)


_fake.keep = []


def _decode_rc(q=(2, 8, 64), kc=(20, 4, 8, 16, 8), vc=(20, 4, 64, 16), w=8, s=0, qd="float16", msl=64, bs=16):
    return _lib.lib.kvc_paged_attention_window(_fake(q, qd), _fake(q, qd), _fake(kc), _fake(vc), _fake((2, 4), "int32"),
                                               _fake((2,), "int32"), 4, 0.125, bs, msl, w, s, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(w=0), 1, "window_size must be positive"),
    (dict(w=-3), 1, "window_size must be positive"),
    (dict(s=-1), 1, "sink_size must be non-negative"),
    (dict(msl=65), 1, "max_seq_len exceeds block table capacity"),
    (dict(qd="int32"), 1, "Unsupported dtype combination"),
    (dict(kc=(20, 4, 8, 8, 8)), 1, "cache block dimensions"),
    (dict(kc=(20, 16, 4, 64), vc=(20, 16, 4, 64), qd="float32"), 4, "float16/bfloat16"),
    (dict(kc=(20, 16), vc=(20, 16)), 1, "key_cache/value_cache must be"),
])
def test_decode_refusals(kw, rc, text):
    assert _decode_rc(**kw) == rc
    assert text in _lib.last_error()


@pytest.mark.parametrize("w,s,text", [(0, 0, "window_size must be positive"), (4, -1, "sink_size must be")])
def test_extend_refusals(w, s, text):
    q = (6, 8, 64)
    rc = _lib.lib.kvc_paged_prefill_window(_fake(q), _fake(q), _fake((20, 4, 8, 16, 8)), _fake((20, 4, 64, 16)),
                                           _fake((2, 4), "int32"), _fake((3,), "int32"), _fake((2,), "int32"), 4, 0.125,
                                           16, 3, w, s, None)
    assert rc == 1 and text in _lib.last_error()
