"""Greedy decoding of a small random decoder with drafts looked up in each sequence's own history, on one GPU.

A step's path through the library: qkv and output projections and the MLP (ak_wq_gemv_kt_multi, ak_wq_gemv_kt_silu), the
new tokens' keys and values into the paged cache (ak_kv_write), attention over it (ak_paged_attn), the int8 LM head
(ak_i8_gemv) and the verification of the drafts (ak_spec_verify).  All of these give a token the same bits whether it comes
alone or beside drafts, so decoding with drafts emits the tokens of decoding without, in fewer steps; the script checks that.
Norms, rotary embedding and residuals are torch's elementwise operations.

    python examples/speculative_decode.py [--bits 16|8|4] [--drafts 4] [--tokens 64]
"""
import argparse
import ctypes
import importlib
import os
import sys
import time

import torch  # before the library: both use torch's HIP runtime

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
L = importlib.import_module("agens-engine_amd").load()

DEV = "cuda"
HIDDEN, HEADS, KV_HEADS, DIM, INTER, LAYERS, VOCAB = 1024, 8, 2, 128, 2048, 2, 2048
GROUP, PAGE = 128, 16
_vp, _i, _l, _f = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float
L.ak_wq_repack_kt.argtypes = [_i, _vp, _vp, _vp, _vp, _i, _i, _i, _vp]
L.ak_wq_kt_weight_bytes.argtypes, L.ak_wq_kt_weight_bytes.restype = [_i, _i, _i], ctypes.c_size_t
L.ak_w4_kt_scale_bytes.argtypes, L.ak_w4_kt_scale_bytes.restype = [_i, _i, _i], ctypes.c_size_t
L.ak_wq_gemv_kt_multi.argtypes = [_i, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp]
L.ak_wq_gemv_kt_silu.argtypes = [_i, _vp, _i, _vp, _vp, _vp, _i, _i, _i, _i, _vp]
L.ak_i8_gemv.argtypes = [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp]
L.ak_kv_page_bytes.argtypes, L.ak_kv_page_bytes.restype = [_i, _i, _i, _i], ctypes.c_size_t
L.ak_kv_write.argtypes = [_i, _vp, _vp, _i, _l, _l, _vp, _vp, _i, _i, _i, _i, _vp]
L.ak_paged_attn.argtypes = [_i, _vp, _i, _l, _vp, _i, _i, _i, _i, _i, _i, _vp, _vp, _vp, _i, _f, _vp, _l, _vp, _vp]
L.ak_spec_verify.argtypes = [_vp, _l, _vp, _l, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp, _vp, _vp]


def check(rc):
    if rc:
        raise RuntimeError(f"error {rc}")


def stream():
    return torch.cuda.current_stream().cuda_stream


class Linear:
    """A 4-bit linear of random weights in the library's layout."""

    def __init__(self, g, n, k):
        self.n, self.k = n, k
        packed = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, k // 8), dtype=torch.int64, generator=g).to(torch.int32).to(DEV)
        scales = ((0.5 + torch.rand((n, k // GROUP), generator=g)) * 0.22 / k ** 0.5).to(torch.bfloat16).to(DEV)
        self.wt = torch.zeros(L.ak_wq_kt_weight_bytes(4, n, k), dtype=torch.uint8, device=DEV)
        self.st = torch.zeros(L.ak_w4_kt_scale_bytes(n, k, GROUP), dtype=torch.uint8, device=DEV)
        check(L.ak_wq_repack_kt(4, packed.data_ptr(), scales.data_ptr(), self.wt.data_ptr(), self.st.data_ptr(), n, k,
                                GROUP, stream()))
        torch.cuda.synchronize()

    def __call__(self, x):
        y = torch.empty((x.shape[0], self.n), dtype=torch.bfloat16, device=DEV)
        one = lambda t: (_vp * 1)(t.data_ptr())
        check(L.ak_wq_gemv_kt_multi(4, x.data_ptr(), x.shape[0], 1, one(self.wt), one(self.st), one(y), (_i * 1)(self.n), None,
                                    self.k, GROUP, 0, stream()))
        return y

    def of_silu(self, gate_up):
        y = torch.empty((gate_up.shape[0], self.n), dtype=torch.bfloat16, device=DEV)
        check(L.ak_wq_gemv_kt_silu(4, gate_up.data_ptr(), gate_up.shape[0], self.wt.data_ptr(), self.st.data_ptr(),
                                   y.data_ptr(), self.n, self.n, self.k, GROUP, stream()))
        return y


class Cache:
    """The pages of one layer; all layers use the same page table."""

    def __init__(self, bits, npages):
        self.bits, self.npages = bits, npages
        self.pool = torch.zeros(npages * L.ak_kv_page_bytes(bits, PAGE, KV_HEADS, DIM), dtype=torch.uint8, device=DEV)

    def write(self, k, v, slots):
        check(L.ak_kv_write(self.bits, k.data_ptr(), v.data_ptr(), len(slots), k.stride(0), v.stride(0), slots.data_ptr(),
                            self.pool.data_ptr(), self.npages, PAGE, KV_HEADS, DIM, stream()))

    def attend(self, q, lens, table):
        y = torch.empty((len(q), HEADS * DIM), dtype=torch.bfloat16, device=DEV)
        check(L.ak_paged_attn(self.bits, q.data_ptr(), len(q), q.stride(0), self.pool.data_ptr(), self.npages, PAGE, HEADS,
                              KV_HEADS, DIM, len(lens), None, lens.data_ptr(), table.data_ptr(), table.shape[1], DIM ** -0.5,
                              y.data_ptr(), HEADS * DIM, None, stream()))
        return y


def norm(x):
    return (x.double() * torch.rsqrt(x.double().pow(2).mean(-1, keepdim=True) + 1e-6)).to(torch.bfloat16)


def rotate(x, pos):
    """Rotary embedding of x [m][heads][DIM] at positions pos."""
    f = 10000.0 ** (-torch.arange(0, DIM, 2, device=DEV, dtype=torch.float64) / DIM)
    a = (pos.double()[:, None] * f)[:, None]
    u, v = x.double().chunk(2, -1)
    return torch.cat([u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin()], -1).to(torch.bfloat16)


class Model:
    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.embed = torch.randn((VOCAB, HIDDEN), generator=g).to(torch.bfloat16).to(DEV)
        self.layers = [(Linear(g, (HEADS + 2 * KV_HEADS) * DIM, HIDDEN), Linear(g, HIDDEN, HEADS * DIM),
                        Linear(g, 2 * INTER, HIDDEN), Linear(g, HIDDEN, INTER)) for _ in range(LAYERS)]
        self.head = torch.randint(-127, 128, (VOCAB, HIDDEN), generator=g, dtype=torch.int8).to(DEV)
        self.head_scale = torch.full((VOCAB,), 0.02 / HIDDEN ** 0.5, device=DEV)

    def __call__(self, tokens, pos, slots, lens, table, caches, head=True):
        """Logits [m][VOCAB] (if `head`) of tokens [m] (each sequence's side by side) at positions pos, cached at slots; lens:
        of the sequences, these tokens included."""
        m = len(tokens)
        x = self.embed[tokens.long()]
        for (qkv, out, gate_up, down), cache in zip(self.layers, caches):
            y = qkv(norm(x)).view(m, HEADS + 2 * KV_HEADS, DIM)
            y[:, :HEADS + KV_HEADS] = rotate(y[:, :HEADS + KV_HEADS], pos)
            cache.write(y[:, HEADS:], y[:, HEADS + KV_HEADS:], slots)
            x = x + out(cache.attend(y[:, :HEADS], lens, table))
            x = x + down.of_silu(gate_up(norm(x)))
        if not head:
            return None
        x = norm(x)
        logits = torch.empty((m, VOCAB), dtype=torch.bfloat16, device=DEV)
        check(L.ak_i8_gemv(x.data_ptr(), self.head.data_ptr(), self.head_scale.data_ptr(), logits.data_ptr(), m, VOCAB, HIDDEN,
                           VOCAB, stream()))
        return logits


def lookup(history, n):
    """Up to n tokens that followed the history's last two where these stood before."""
    for i in range(len(history) - 3, -1, -1):
        if history[i:i + 2] == history[-2:]:
            return history[i + 2:i + 2 + n]
    return []


def decode(model, prompts, count, drafts, bits):
    """The first `count` tokens after each prompt, and the steps this took."""
    b, t = len(prompts), drafts
    need = (max(map(len, prompts)) + count + 2 * t + 2 + PAGE - 1) // PAGE
    table = torch.randperm(b * need, device=DEV).to(torch.int32).view(b, need)
    caches = [Cache(bits, b * need) for _ in range(LAYERS)]

    def forward(tokens, first, head=True):  # tokens [b][n], the first of each at position first[i]
        n = len(tokens[0])
        pos = torch.tensor([p + j for p in first for j in range(n)], dtype=torch.int32, device=DEV)
        seq = torch.arange(b, device=DEV).repeat_interleave(n)
        slots = table[seq, (pos // PAGE).long()] * PAGE + pos % PAGE
        lens = torch.tensor([p + n for p in first], dtype=torch.int32, device=DEV)
        flat = torch.tensor(tokens, dtype=torch.int32, device=DEV).reshape(-1)
        return model(flat, pos, slots, lens, table, caches, head)

    history = [list(p) for p in prompts]
    forward([h[:-1] for h in history], [0] * b, head=False)  # (prompts of one length, all but the last token in one call)
    done = [len(h) - 1 for h in history]  # tokens in the cache
    u = torch.zeros((b, t + 1), device=DEV)
    cold = torch.zeros((b,), device=DEV)  # greedy
    emitted = torch.empty((b, t + 1), dtype=torch.int32, device=DEV)
    accepted = torch.empty((b,), dtype=torch.int32, device=DEV)
    steps = 0
    while min(len(h) - len(p) for h, p in zip(history, prompts)) < count:
        drafted = [lookup(h, t) if t and len(h) - len(p) < count else [] for h, p in zip(history, prompts)]
        counts = torch.tensor([len(d) for d in drafted], dtype=torch.int32, device=DEV)
        padded = [d + [0] * (t - len(d)) for d in drafted]
        logits = forward([[h[-1]] + d for h, d in zip(history, padded)], done)
        ids = torch.tensor(padded, dtype=torch.int32, device=DEV).reshape(b, t)
        check(L.ak_spec_verify(logits.data_ptr(), VOCAB, None, 0, ids.data_ptr() if t else None, counts.data_ptr(),
                               u.data_ptr(), cold.data_ptr(), b, t, VOCAB, emitted.data_ptr(), accepted.data_ptr(), None,
                               stream()))
        for i, (row, n) in enumerate(zip(emitted.tolist(), accepted.tolist())):
            if len(history[i]) - len(prompts[i]) < count:  # (a sequence that is done stays where it is)
                history[i] += row[:n + 1]
                done[i] += n + 1
        steps += 1
    return [h[len(p):len(p) + count] for h, p in zip(history, prompts)], steps


def main():
    a = argparse.ArgumentParser()
    a.add_argument("--bits", type=int, default=8, choices=(16, 8, 4))
    a.add_argument("--drafts", type=int, default=4)
    a.add_argument("--tokens", type=int, default=64)
    a = a.parse_args()
    model = Model(1)
    prompts = [[5, 17, 99, 3, 250, 17, 99, 3], [1, 2, 3, 4, 1, 2, 3, 4], [900, 30, 7, 61, 44, 2, 8, 1000]]
    result = {}
    for t in (0, a.drafts):
        decode(model, prompts, 4, t, a.bits)
        start = time.perf_counter()
        result[t] = decode(model, prompts, a.tokens, t, a.bits)
        print(f"drafts {t}: {result[t][1]} steps for {a.tokens} tokens of {len(prompts)} sequences, "
              f"{time.perf_counter() - start:.2f} s", flush=True)
    if result[0][0] != result[a.drafts][0]:
        raise SystemExit("the tokens differ")
    print("the same tokens")


if __name__ == "__main__":
    main()
