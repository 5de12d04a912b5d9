"""Serving a sliding-window model's attention layers from one paged KV cache.

Requests arrive over time with prompts of different lengths.  Every step takes a
chunk of each unfinished prompt and one token of each running request, and runs

    build_step_tables      once per step: block tables, positions, cache slots
    qk_norm_rope_append    per layer: q / k norms, rotary position, cache append
    paged_prefill_window   per layer, steps that bring more than one token somewhere
    paged_attention_window per layer, steps of one token per request

Blocks that have left every window (and hold no sink) go back to the free list, so
a request of any length holds a bounded number of them.  The projections around the
attention are random numbers here; the attention of every step is checked against
the formula in float64.

    python examples/window_serving.py [--steps N] [--requests B]
"""

import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "sglang-mlx_b200"))

from sglang_mlx_b200 import metal_kernels as mk  # noqa: E402
from sglang_mlx_b200.device_array import DeviceArray  # noqa: E402

HEADS, KV_HEADS, DIM, BLOCK = 8, 2, 64, 16
WINDOW, SINKS, CHUNK, LAYERS = 96, 4, 40, 2
SCALE, EPS, BASE = DIM ** -0.5, 1e-6, 10000.0


class Engine:
    """The device state of the layers, and the host's view of requests and blocks."""

    def __init__(self, max_requests, max_len, num_blocks, seed=0):
        rng = np.random.default_rng(seed)
        self.rng, self.max_len = rng, max_len
        self.rope = mk.rotary_table(max_len, DIM, BASE)
        self.tables = DeviceArray.from_numpy(np.full((max_requests, -(-max_len // BLOCK)), -1, np.int32))
        self.lens = np.zeros(max_requests, np.int32)
        self.host_tables = [[] for _ in range(max_requests)]  # block ids by block index, None once freed
        self.free = list(rng.permutation(num_blocks))
        self.k_cache = [DeviceArray.zeros((num_blocks, KV_HEADS, DIM // 8, BLOCK, 8), "float16") for _ in range(LAYERS)]
        self.v_cache = [DeviceArray.zeros((num_blocks, KV_HEADS, DIM, BLOCK), "float16") for _ in range(LAYERS)]
        self.q_w = [(1 + 0.1 * rng.standard_normal(DIM)).astype(np.float16) for _ in range(LAYERS)]
        self.k_w = [(1 + 0.1 * rng.standard_normal(DIM)).astype(np.float16) for _ in range(LAYERS)]
        # what the check needs: every token's raw keys and values, by layer and request
        self.keys = [[np.zeros((0, KV_HEADS, DIM)) for _ in range(max_requests)] for _ in range(LAYERS)]
        self.values = [[np.zeros((0, KV_HEADS, DIM)) for _ in range(max_requests)] for _ in range(LAYERS)]

    def step(self, new):
        """One step of new[b] tokens for request b; returns the largest error of any layer's output."""
        new = np.asarray(new, np.int32)
        need = [-(-int(n + m) // BLOCK) - len(t) for n, m, t in zip(self.lens, new, self.host_tables)]
        t = mk.build_step_tables(self.tables, self.lens, new, np.asarray(self.free[:max(1, sum(need))], np.int32), BLOCK)
        for row, n in zip(self.host_tables, need):  # the same blocks, in request order
            row.extend(self.free[:n])
            del self.free[:n]
        prefix, self.lens = self.lens, self.lens + new
        tokens, worst = int(new.sum()), 0.0
        for layer in range(LAYERS):
            q, k, v = (self.rng.standard_normal((tokens, h, DIM)).astype(np.float16) for h in (HEADS, KV_HEADS, KV_HEADS))
            k_cache, v_cache = self.k_cache[layer], self.v_cache[layer]
            qd, _, _ = mk.qk_norm_rope_append(q, k, v, t.positions, self.rope, k_cache, v_cache, t.slot_mapping,
                                              q_weight=self.q_w[layer], k_weight=self.k_w[layer], eps=EPS)
            if new.max() == 1 and new.min() == 1:
                out = mk.paged_attention_window(qd, k_cache, v_cache, self.tables, t.kv_lens, KV_HEADS, SCALE, BLOCK,
                                                self.max_len, WINDOW, SINKS)
            else:
                out = mk.paged_prefill_window(qd, k_cache, v_cache, self.tables, t.qo_indptr, t.kv_lens, KV_HEADS, SCALE,
                                              BLOCK, WINDOW, SINKS, max_q_len=int(new.max()))
            worst = max(worst, self.check(layer, prefix, new, q, k, v, out.to_numpy()))
        self.release()
        return worst

    def release(self):
        """Blocks behind the window, past the sinks, are free for anyone."""
        for row, n in zip(self.host_tables, self.lens):
            for i in range(-(-SINKS // BLOCK), max(0, int(n) + 1 - WINDOW) // BLOCK):
                if row[i] is not None:
                    self.free.append(row[i])
                    row[i] = None

    def check(self, layer, prefix, new, q, k, v, out):
        at, worst = 0, 0.0
        for b, m in enumerate(new):
            rows = slice(at, at + int(m))
            at += int(m)
            pos = int(prefix[b]) + np.arange(int(m))
            kr = rotate(k[rows], self.k_w[layer], pos).astype(np.float16).astype(np.float64)  # as it is cached
            self.keys[layer][b] = K = np.concatenate([self.keys[layer][b], kr])
            self.values[layer][b] = V = np.concatenate([self.values[layer][b], v[rows].astype(np.float64)])
            qr = rotate(q[rows], self.q_w[layer], pos).astype(np.float16).astype(np.float64)
            for i, p in enumerate(pos):
                j = np.arange(p + 1)
                j = j[(j < SINKS) | (j > p - WINDOW)]
                for h in range(HEADS):
                    s = K[j, h * KV_HEADS // HEADS] @ qr[i, h] * SCALE
                    w = np.exp(s - s.max())
                    want = w @ V[j, h * KV_HEADS // HEADS] / w.sum()
                    worst = max(worst, float(np.abs(out[rows][i, h].astype(np.float64) - want).max()))
        return worst


def rotate(x, weight, pos):
    """RMS norm with a weight, then the rotary position, in float64."""
    x = x.astype(np.float64)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * weight.astype(np.float64)
    f, _ = mk.rotary_frequencies(DIM, BASE)
    a = pos[:, None, None] * f
    lo, hi = x[..., :DIM // 2], x[..., DIM // 2:]
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], -1)


def main(steps=30, requests=4, seed=0, log=print):
    rng = np.random.default_rng(seed)
    prompts = rng.integers(1, 300, requests)
    arrives = np.sort(rng.integers(0, 4, requests))
    arrives[0] = 0
    bound = requests * (-(-(WINDOW + CHUNK) // BLOCK) + 3)  # blocks that the requests can hold at one time
    eng = Engine(requests, int(prompts.max()) + steps + 1, bound, seed)
    worst = 0.0
    for s in range(steps):
        left = np.where(arrives <= s, np.maximum(prompts - eng.lens, 0), 0)
        new = np.where(left > 0, np.minimum(left, CHUNK), (arrives <= s).astype(np.int64))
        err = eng.step(new)
        worst = max(worst, err)
        log(f"step {s:2d}: new tokens {new.tolist()}, lengths {eng.lens.tolist()}, blocks free {len(eng.free)}/{bound}, "
            f"largest error {err:.1e}")
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--requests", type=int, default=4)
    a = ap.parse_args()
    worst = main(a.steps, a.requests)
    print(f"largest error of any output: {worst:.1e}")
    # values of at most about 4.5, a few roundings to 11 bits on the way
    sys.exit(0 if worst < 8.8e-3 else 1)
