"""Requests of unequal length with adapters and sampling settings of their own, served in one batch of a small random decoder on
one GPU: new ones join as others end.

A step's path through the library: the batch's pages, positions and slots (ak_kv_plan), the tokens grouped by adapter
(ak_lora_plan), then per layer the qkv projection and its adapters (ak_wq_gemv_kt_multi, ak_lora_add), rotary positions on the
way into the paged cache (ak_rope_kv_write), attention over it (ak_paged_attn), output projection and MLP, and after the int8 LM
head (ak_i8_gemv) the next tokens (ak_sample).  Running requests take one token a step, new ones their whole prompt.  All of
these give a token the same bits whatever else is in the call, so a request gets the same tokens in a batch as alone; the script
checks that.  Norms and residuals are torch's elementwise operations.

    python examples/batched_serving.py [--bits 16|8|4] [--requests 9] [--rows 4]
"""
import argparse
import ctypes
import random
import time

import torch

from speculative_decode import (DEV, DIM, HEADS, HIDDEN, INTER, KV_HEADS, LAYERS, PAGE, VOCAB, Cache, L, Linear, check, norm,
                                stream)

_vp, _i, _l, _f = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float
L.ak_kv_plan.argtypes = [_i, _i] + [_vp] * 6 + [_i, _i, _vp, _i] + [_vp] * 8
L.ak_rope_freqs.argtypes = [ctypes.c_double, _i, _i, ctypes.c_double, _l, ctypes.c_double, ctypes.c_double, _vp, _vp]
L.ak_rope_kv_write.argtypes = [_i, _vp, _l, _vp, _l, _vp, _l, _vp, _l, _i, _i, _vp, _vp, _i, _i, _f, _vp, _vp] + [_i] * 4 + [_vp]
L.ak_lora_plan_bytes.argtypes, L.ak_lora_plan_bytes.restype = [_i, _i, _i, _i], ctypes.c_size_t
L.ak_lora_plan.argtypes = [_vp, _i, _i, _vp, _vp]
L.ak_lora_add.argtypes = [_vp, _vp, _i, _l, _i, _i, _i, _vp, _vp, _i] + [_vp] * 5 + [_vp]
L.ak_sample.argtypes = [_vp, _l, _vp, _vp, _vp, _vp, _vp, _i, _i, _vp, _vp, _vp]

ADAPTERS, RANK, MOST = 3, 16, 128  # MOST: tokens of a step
WIDTHS = [HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM]


def _p(t):
    return t.data_ptr()


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32, device=DEV)


class Model:
    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        small = lambda *s: (torch.randn(s, generator=g) * s[-1] ** -0.5).to(torch.bfloat16).to(DEV)  # noqa: E731
        self.embed = torch.randn((VOCAB, HIDDEN), generator=g).to(torch.bfloat16).to(DEV)
        self.layers = [(Linear(g, sum(WIDTHS), HIDDEN), Linear(g, HIDDEN, HEADS * DIM), Linear(g, 2 * INTER, HIDDEN),
                        Linear(g, HIDDEN, INTER)) for _ in range(LAYERS)]
        self.down = [small(ADAPTERS, 3 * RANK, HIDDEN) for _ in range(LAYERS)]
        self.up = [[small(ADAPTERS, n, RANK) for n in WIDTHS] for _ in range(LAYERS)]
        self.head = torch.randint(-127, 128, (VOCAB, HIDDEN), generator=g, dtype=torch.int8).to(DEV)
        self.head_scale = torch.full((VOCAB,), 0.06 / HIDDEN ** 0.5, device=DEV)
        f, mag = torch.zeros(DIM // 2, dtype=torch.float64), ctypes.c_float(0)
        check(L.ak_rope_freqs(10000.0, DIM, 0, 1.0, 0, 0.0, 0.0, _p(f), ctypes.byref(mag)))
        self.freqs, self.mag = f.to(DEV), mag.value
        self.plan = torch.zeros(L.ak_lora_plan_bytes(MOST, ADAPTERS, 3 * RANK, HIDDEN), dtype=torch.uint8, device=DEV)


class Server:
    """`rows` sequences at most, with all the state of the batch on the GPU."""

    def __init__(self, model, bits, rows, room=128):
        self.model, self.bits, self.rows, self.ldt = model, bits, rows, room // PAGE
        self.npages = rows * self.ldt
        self.caches = [Cache(bits, self.npages) for _ in range(LAYERS)]
        self.table, self.free = _i32(rows, self.ldt), torch.randperm(self.npages, device=DEV).to(torch.int32)
        self.nfree = torch.full((1,), self.npages, dtype=torch.int32, device=DEV)
        self.cached, self.held, self.refused, self.qstart = _i32(rows), _i32(rows), _i32(rows), _i32(rows + 1)

    def step(self, tokens, counts, drop, adapter, settings):
        """The next token of every row that has new ones.  tokens: of the rows, side by side."""
        md, b, m = self.model, self.rows, len(tokens)
        one = lambda t: torch.tensor(t, dtype=torch.int32, device=DEV)  # noqa: E731
        tokens, counts, drop, adapter = one(tokens), one(counts), one(drop), one(adapter)
        pos, slots = _i32(m), _i32(m)
        check(L.ak_kv_plan(b, m, _p(counts), _p(drop), _p(self.cached), _p(self.held), _p(self.nfree), _p(self.free),
                           self.npages, PAGE, _p(self.table), self.ldt, _p(self.cached), _p(self.held), _p(self.nfree),
                           _p(self.qstart), _p(pos), _p(slots), _p(self.refused), stream()))
        lens = self.cached
        ids = torch.repeat_interleave(adapter, counts, output_size=m)
        check(L.ak_lora_plan(_p(ids), m, ADAPTERS, _p(md.plan), stream()))
        x = md.embed[tokens.long()]
        width = sum(WIDTHS)
        for (qkv, out, gate_up, down), a, up, cache in zip(md.layers, md.down, md.up, self.caches):
            h = norm(x)
            y = qkv(h)
            ptrs = lambda ts: (_vp * 3)(*ts)  # noqa: E731
            at = [_p(y), _p(y) + 2 * WIDTHS[0], _p(y) + 2 * (WIDTHS[0] + WIDTHS[1])]  # q, k and v within a row
            check(L.ak_lora_add(_p(md.plan), _p(h), m, HIDDEN, HIDDEN, ADAPTERS, RANK, _p(a), None, 3, ptrs(map(_p, up)), None,
                                ptrs(at), (_i * 3)(*WIDTHS), (_i * 3)(width, width, width), stream()))
            check(L.ak_rope_kv_write(self.bits, at[0], width, at[1], width, at[2], width, at[0], width, m, HEADS, _p(pos),
                                     _p(md.freqs), DIM, 0, md.mag, _p(slots), _p(cache.pool), self.npages, PAGE, KV_HEADS, DIM,
                                     stream()))
            att = torch.empty((m, HEADS * DIM), dtype=torch.bfloat16, device=DEV)
            check(L.ak_paged_attn(self.bits, at[0], m, width, _p(cache.pool), self.npages, PAGE, HEADS, KV_HEADS, DIM, b,
                                  _p(self.qstart), _p(lens), _p(self.table), self.ldt, DIM ** -0.5, _p(att), HEADS * DIM, None,
                                  stream()))
            x = x + out(att)
            x = x + down.of_silu(gate_up(norm(x)))
        last = norm(x[(self.qstart[1:].long() - 1).clamp(min=0)])  # of rows without new tokens: not used
        logits = torch.empty((b, VOCAB), dtype=torch.bfloat16, device=DEV)
        for i in range(0, b, 16):
            check(L.ak_i8_gemv(_p(last[i:]), _p(md.head), _p(md.head_scale), _p(logits[i:]), min(16, b - i), VOCAB, HIDDEN, VOCAB,
                               stream()))
        heat, top_k, top_p, min_p, u = (torch.tensor(v, device=DEV) for v in zip(*settings))
        top_k, picked = top_k.to(torch.int32), _i32(b)
        check(L.ak_sample(_p(logits), VOCAB, _p(heat), _p(top_k), _p(top_p), _p(min_p), _p(u), b, VOCAB, _p(picked), None,
                          stream()))
        if int(self.refused.sum()):
            raise RuntimeError("out of pages")
        return picked.tolist()


class Request:
    def __init__(self, seed):
        rng = random.Random(seed)
        self.prompt = [rng.randrange(VOCAB) for _ in range(rng.randint(1, 20))]
        self.adapter = rng.randint(-1, ADAPTERS - 1)
        self.count = rng.randint(5, 40)
        self.settings = (rng.choice([0.0, 0.7, 1.0, 1.3]), rng.choice([0, 5, 50]), rng.choice([1.0, 0.9, 0.6]),
                         rng.choice([0.0, 0.02]))
        self.u = [rng.random() for _ in range(self.count)]


def serve(model, bits, requests, rows):
    """Every request's tokens, and the steps this took."""
    server = Server(model, bits, rows)
    waiting, running, done = list(enumerate(requests)), [None] * rows, {}
    given = [[] for _ in requests]
    ended, steps = [0] * rows, 0
    while waiting or any(running):
        tokens, counts, adapter, settings = [], [], [], []
        for i in range(rows):
            if running[i] is None and waiting and len(tokens) + len(waiting[0][1].prompt) + rows <= MOST:
                running[i] = waiting.pop(0)
            if running[i] is None:
                counts.append(0)
                adapter.append(-1)
                settings.append((0.0, 0, 1.0, 0.0, 0.0))
                continue
            j, r = running[i]
            new = r.prompt if not given[j] else given[j][-1:]
            tokens += new
            counts.append(len(new))
            adapter.append(r.adapter)
            settings.append(r.settings + (r.u[len(given[j])],))
        picked = server.step(tokens, counts, ended, adapter, settings)
        ended = [0] * rows
        steps += 1
        for i in range(rows):
            if running[i] is None:
                continue
            j, r = running[i]
            given[j].append(picked[i])
            if len(given[j]) == r.count:  # its pages go back with the next step, whoever takes the row
                done[j], running[i], ended[i] = given[j], None, 1
    return [done[j] for j in range(len(requests))], steps


def main():
    a = argparse.ArgumentParser()
    a.add_argument("--bits", type=int, default=8, choices=(16, 8, 4))
    a.add_argument("--requests", type=int, default=9)
    a.add_argument("--rows", type=int, default=4)
    a = a.parse_args()
    model, requests = Model(1), [Request(s) for s in range(a.requests)]
    start = time.perf_counter()
    together, steps = serve(model, a.bits, requests, a.rows)
    print(f"{a.requests} requests, {sum(map(len, together))} tokens in {steps} steps of up to {a.rows} rows, "
          f"{time.perf_counter() - start:.2f} s", flush=True)
    for j, r in enumerate(requests):
        alone, _ = serve(model, a.bits, [r], 1)
        if alone[0] != together[j]:
            raise SystemExit(f"request {j}: the tokens differ")
    print("the same tokens alone")


if __name__ == "__main__":
    main()
