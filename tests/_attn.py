"""Attention over the cache against 64 bits, with a tolerance that follows each key's own share.  Test infrastructure.

What the definition leaves to the kernel's arithmetic, all of it fp32 (u = 2^-24; the matrix unit's sums may drop bits instead
of rounding them, so 2u a step there):
  a score      is a sum of 2 dim products, the codes' and their offset's (dim in bf16), and some factors:
               dz_j = (2 dim + 8) * 2u * scale * s_j * sum |q| (|code_j| + offset);
  a weight     exp(z_j - top): the two products' roundings and the exponential's own, ez_j = (|z_j| + |top| + 2) * 2^-22;
  an output    sum w_j v_j / sum w_j: each weight's error moves it by p_j (dz_j + ez_j) |v_j - y|; the weights beside the values
               keep 16 bits at least, their sums take a step for each of a part's 128 tokens, 8 parts, 16 blocks and the
               context's groups of blocks: (2^-16 + steps * 2u) sum p |v|; then its own rounding, half of bf16's last place;
  lse          sum p_j (dz_j + ez_j), a step u for each of a lane's 32 tokens of a part, parts, blocks and groups, its rounding."""
import types

import numpy as np

from _lib import f2bf_array, bf2f_array
from _ops import ops, page_bytes, quantise
from test_gpu_paged_attn import Batch

U = 2.0 ** -24


def bf16(x):
    x = np.asarray(x, dtype=np.float32)
    return f2bf_array(x.ravel()).reshape(x.shape)


class Held:
    """Keys or values [n][kv][dim] (bf16 bits) as the cache holds them: values and, for the error, sum of what is multiplied."""

    def __init__(self, x, bits):
        self.bits = bits
        if bits == 16:
            self.x = bf2f_array(x).astype(np.float64)
            self.most = np.abs(self.x)
        else:
            c, s = quantise(x, bits)
            off, s = 128 if bits == 8 else 8, bf2f_array(s).astype(np.float64)[..., None]
            c = c.astype(np.float64) - off
            self.x, self.most = c * s, (np.abs(c) + off) * s


class Scene(Batch):
    """Sequences with their pages, made at once (contexts of tens of thousands of tokens).  sharp: size of the queries."""

    def __init__(self, seed, bits, page, heads, kv, dim, lens, counts, sharp=1.0, spare=2, vsize=None, ldt=None):
        rng = self.rng = np.random.default_rng(seed)
        self.bits, self.page, self.heads, self.kv, self.dim = bits, page, heads, kv, dim
        self.lens, self.counts = list(lens), list(counts)
        self.m, self.b = sum(counts), len(lens)
        need = [(n + page - 1) // page for n in lens]
        self.npages = sum(need) + spare
        self.ldt = ldt or max(need + [1]) + 1
        self.table = np.full((self.b, self.ldt), -7, dtype=np.int32)
        order, at = rng.permutation(self.npages), 0
        self.mem = np.full((self.npages, page_bytes(bits, page, kv, dim)), 0xFF, dtype=np.uint8)
        self.k, self.v, self.present = [], [], []
        for i, n in enumerate(lens):
            self.table[i, :need[i]] = order[at:at + need[i]]
            at += need[i]
            k, v = (rng.standard_normal((n, kv, dim), dtype=np.float32) for _ in range(2))
            if vsize is not None:
                v *= vsize(i, n)[:, None, None].astype(np.float32)
            self.k.append(bf16(k)), self.v.append(bf16(v))
            self.present.append(np.ones(n, dtype=bool))
        self.q = bf16(rng.standard_normal((self.m, heads, dim)) * sharp)
        self.scale = dim ** -0.5
        self.first = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.fill()

    def fill(self):
        """The pages' bytes by the documented layout."""
        rb, plane = self.dim * self.bits // 8, self.page * self.dim * self.bits // 8
        rows = self.mem[:, :2 * self.kv * plane].reshape(self.npages, self.kv, 2, self.page, rb)
        for i, n in enumerate(self.lens):
            pg, off = self.table[i, np.arange(n) // self.page], np.arange(n) % self.page
            for part, x in ((0, self.k[i]), (1, self.v[i])):
                if self.bits == 16:
                    rows[pg, :, part, off] = x.view(np.uint8).reshape(n, self.kv, rb)
                    continue
                c, s = quantise(x, self.bits)
                rows[pg, :, part, off] = c if self.bits == 8 else c[..., 0::2] | (c[..., 1::2] << 4)
                at = 2 * self.kv * plane
                sc = self.mem[:, at:at + self.kv * self.page * 4].reshape(self.npages, self.kv, self.page, 2, 2)
                sc[pg, :, off, part] = s.view(np.uint8).reshape(n, self.kv, 2)

    def device(self):
        self.pool = types.SimpleNamespace(mem=self.mem)  # (where Batch.device looks for them)
        return super().device()

    def expect(self):
        """y, its tolerance, lse, its tolerance."""
        m, h, d, g = self.m, self.heads, self.dim, self.heads // self.kv
        y, ty = np.zeros((m, h, d)), np.zeros((m, h, d))
        lse, tl = np.full((m, h), -np.inf), np.zeros((m, h))
        q = bf2f_array(self.q).astype(np.float64)
        for i, n in enumerate(self.lens):
            held = Held(self.k[i], self.bits), Held(self.v[i], self.bits)
            t = self.counts[i]
            for a in range(h):
                k, kmost, v = held[0].x[:, a // g], held[0].most[:, a // g], held[1].x[:, a // g]
                for j in range(t):
                    use = np.flatnonzero(self.present[i][:max(0, n - t + j + 1)])
                    if not len(use):
                        continue
                    r = self.first[i] + j
                    z = k[use] @ q[r, a] * self.scale
                    top = z.max()
                    e = np.exp(z - top)
                    p = e / e.sum()
                    dz = (2 * d + 8) * 2 * U * abs(self.scale) * (kmost[use] @ np.abs(q[r, a]))
                    err = p * (dz + (np.abs(z) + abs(top) + 2) * 2.0 ** -22)
                    y[r, a], lse[r, a] = p @ v[use], top + np.log(e.sum())
                    steps = 128 + 8 + 16 + len(use) / 16384
                    mag = p @ np.abs(v[use])
                    off = (2.0 ** -16 + steps * 2 * U) * mag + err @ np.abs(v[use]) + err.sum() * np.abs(y[r, a])
                    ty[r, a] = off + np.ldexp(1.0, np.maximum(np.frexp(np.abs(y[r, a]) + off)[1], -125) - 9)
                    tl[r, a] = err.sum() + (32 + 8 + 16 + 8 + len(use) / 16384) * U + 2.0 ** -22 * (1 + abs(lse[r, a]))
        return y, ty, lse, tl

    def compare(self, y, e, rows=slice(None)):
        wy, ty, wl, tl = self.expect()
        off = np.abs(bf2f_array(y).astype(np.float64) - wy) / np.where(ty > 0, ty, 1)
        empty = np.isneginf(wl)
        assert np.array_equal(np.isneginf(e)[rows], empty[rows]) and not y[empty].any()
        assert (off[rows] <= 1).all(), f"{(~(off[rows] <= 1)).sum()} of {off[rows].size} outputs, worst {off[rows].max():.2f}"
        el = np.abs(np.where(empty, 0, e) - np.where(empty, 0, wl)) / np.where(tl > 0, tl, 1)
        assert (el[rows] <= 1).all(), f"lse: {(~(el[rows] <= 1)).sum()} of {el[rows].size}, worst {el[rows].max():.2f}"
        return float(np.nanmax(off[rows], initial=0)), float(np.nanmax(el[rows], initial=0))
