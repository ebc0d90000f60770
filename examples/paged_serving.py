"""Continuous batching over a paged KV cache with the library's operators.

A stack of attention layers (INT8 projections as `QT` weights, fp32
activations, bf16 cache; grouped heads, sinks, every other layer with a
sliding window) serves requests that join as others end.  Each step:

  kv_tables                 pages and slots of the step, on the device
  per layer  QT.matmul      q, k, v of the step's rows
             kv_store       k and v to their slots
             Attention      .packed while all rows are whole prompts, else
                            .paged (chunks of prompts beside single tokens)
             QT.matmul      the output projection, added to the rows

Every request's final rows are then compared with the same layers run over
its whole sequence at once.  Usage: python examples/paged_serving.py
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from picchio_b200 import FMT_INT8, QT, Attention, kv_store, kv_tables  # noqa: E402
from picchio_b200.synth import quantize_int8  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, LAYERS, WINDOW = 256, 16, 2, 64, 2, 48
PAGE, SLOTS, ROWS, CHUNK = 16, 6, 160, 96  # positions a page, requests at a time, rows a step, prompt rows of one request


class Layer:
    def __init__(self, rng, index, pages):
        width = (HEADS + 2 * KV_HEADS) * DIM
        self.qkv = self._weight(rng, width, HIDDEN, 3.0)
        self.out = self._weight(rng, HIDDEN, HEADS * DIM, 0.3)
        self.sinks = torch.from_numpy(rng.standard_normal(HEADS).astype(np.float32)).cuda()
        self.window = WINDOW if index % 2 else 0
        shape = (pages, PAGE, KV_HEADS, DIM)
        # what a page holds before it is written takes no part in anything
        self.k = torch.full(shape, float("nan"), dtype=torch.bfloat16, device="cuda")
        self.v = torch.full(shape, float("nan"), dtype=torch.bfloat16, device="cuda")

    @staticmethod
    def _weight(rng, rows, cols, scale):
        q, s = quantize_int8((rng.standard_normal((rows, cols)) * scale / cols ** 0.5).astype(np.float32))
        return QT(FMT_INT8, rows, cols, q, s)

    def project(self, x):
        """q, k, v of the rows of x, as slices of one product's rows."""
        y = self.qkv.matmul(x).view(-1, HEADS + 2 * KV_HEADS, DIM)
        return y[:, :HEADS].bfloat16(), y[:, HEADS:HEADS + KV_HEADS], y[:, HEADS + KV_HEADS:]


def serve(requests, pages, seed=0, log=print):
    """Serves (prompt length, tokens to add) requests; returns for each its
    input rows, the final rows of all its positions, and the layers."""
    rng = np.random.default_rng(seed)
    layers = [Layer(rng, i, pages) for i in range(LAYERS)]
    inputs = [torch.from_numpy(rng.standard_normal((p + n, HIDDEN)).astype(np.float32)).cuda() for p, n in requests]
    results = [torch.zeros_like(x) for x in inputs]
    attention = Attention()

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    longest = max(p + n for p, n in requests)
    page_table = torch.full((SLOTS, -(-longest // PAGE)), -1, dtype=torch.int32, device="cuda")
    free, n_free = torch.arange(pages, dtype=torch.int32, device="cuda"), ints([pages])
    kv_len = ints([0] * SLOTS)
    slot = [None] * SLOTS  # the request in each slot
    done = [0] * len(requests)
    waiting = list(range(len(requests)))
    steps = {"packed": 0, "paged": 0, "refused": 0}
    while waiting or any(r is not None for r in slot):
        new = [0] * SLOTS
        for s in range(SLOTS):
            if slot[s] is None and waiting:
                slot[s] = waiting.pop(0)
            if slot[s] is not None:
                prompt, more = requests[slot[s]]
                left = prompt - done[slot[s]]
                new[s] = min(left, CHUNK) if left > 0 else 1 if done[slot[s]] < prompt + more else -1
        t = kv_tables(kv_len, ints(new), page_table, free, n_free, page_size=PAGE, n_tokens=ROWS)
        kv_len, n_free = t.kv_len, t.n_free
        cu, served = t.cu_new.tolist(), t.served.tolist()
        fresh = all(done[slot[s]] == 0 for s in range(SLOTS) if served[s] and new[s] > 0)
        x = torch.zeros(ROWS, HIDDEN, device="cuda")
        for s in range(SLOTS):
            if served[s] and new[s] > 0:
                x[cu[s]:cu[s + 1]] = inputs[slot[s]][done[slot[s]]:done[slot[s]] + new[s]]
        if cu[-1] == 0 and not any(n < 0 for n in new):
            raise RuntimeError("no request can be served: too few pages")
        if cu[-1]:
            for layer in layers:
                q, k, v = layer.project(x)
                kv_store(layer.k, layer.v, k, v, t.slots)
                a = torch.zeros(ROWS, HEADS, DIM, dtype=torch.bfloat16, device="cuda")  # rows past the step's stay zero
                if fresh:
                    attention.packed(q, k.bfloat16(), v.bfloat16(), t.cu_new, sinks=layer.sinks, window=layer.window, out=a)
                else:
                    attention.paged(q, layer.k, layer.v, page_table, t.cu_new, kv_len, sinks=layer.sinks,
                                    window=layer.window, out=a)
                x = x + layer.out.matmul(a.float().view(ROWS, HEADS * DIM))
            steps["packed" if fresh else "paged"] += 1
        for s in range(SLOTS):
            r = slot[s]
            if r is None or new[s] == 0:
                continue
            if new[s] < 0:
                slot[s] = None  # its pages are back
            elif served[s]:
                results[r][done[r]:done[r] + new[s]] = x[cu[s]:cu[s + 1]]
                done[r] += new[s]
            else:
                steps["refused"] += 1  # comes again when pages or rows are there
    attention.check()
    log(f"{len(requests)} requests, {sum(p + n for p, n in requests)} positions, {pages} pages: {steps}")
    assert int(n_free) == pages, "pages are missing"
    return inputs, results, layers, steps


def whole(x, layers):
    """The same layers over one sequence at once: dense attention in fp64."""
    n = x.shape[0]
    at = torch.arange(n, device="cuda")
    for layer in layers:
        q, k, v = layer.project(x)
        hidden = at[None] > at[:, None]
        if layer.window:
            hidden |= at[None] <= at[:, None] - layer.window
        group = HEADS // KV_HEADS
        k, v = (y.bfloat16().double().repeat_interleave(group, 1) for y in (k, v))
        z = torch.einsum("qhd,khd->hqk", q.double(), k) * DIM ** -0.5
        z = z.masked_fill(hidden, float("-inf"))
        sink = layer.sinks.double().view(HEADS, 1, 1).expand(HEADS, n, 1)
        w = torch.softmax(torch.cat([z, sink], 2), 2)[..., :n]
        a = torch.einsum("hqk,khd->qhd", w, v).bfloat16().float()
        x = x + layer.out.matmul(a.reshape(n, HEADS * DIM))
    return x


def main(log=print):
    requests = [(40, 9), (7, 30), (130, 4), (1, 12), (64, 20), (200, 1), (33, 40), (16, 16), (90, 3), (5, 5)]
    inputs, results, layers, steps = serve(requests, pages=40, log=log)
    worst = 0.0
    for x, got in zip(inputs, results):
        want = whole(x, layers)
        worst = max(worst, float((got - want).norm() / (want - x).norm()))
    log(f"largest relative difference from the whole sequences: {worst:.2e}")
    # bf16 weights and attention outputs: a few units of 2^-9 a layer
    if worst > 2e-2:
        raise SystemExit("the served rows differ from the whole sequences'")
    return steps, worst


if __name__ == "__main__":
    main()
