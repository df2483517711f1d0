"""Bindings and 64-bit restatements (numpy) of the operators between the linears: the paged key-value cache, attention over
it and the verification of drafts.  Test infrastructure: the oracle."""
import ctypes

import numpy as np

from _lib import kernels, c_void_p, bf2f_array, f2bf_array

_i, _l, _vp, _f = ctypes.c_int, ctypes.c_long, c_void_p, ctypes.c_float
_bound = None


def ops():
    global _bound
    if _bound is None:
        K = kernels()
        K.ak_kv_page_bytes.restype, K.ak_kv_page_bytes.argtypes = ctypes.c_size_t, [_i] * 4
        K.ak_kv_write.argtypes = [_i, _vp, _vp, _i, _l, _l, _vp, _vp, _i, _i, _i, _i, _vp]
        K.ak_kv_read.argtypes = [_i, _vp, _i, _i, _i, _i, _vp, _i, _vp, _vp, _l, _l, _vp]
        K.ak_paged_attn.argtypes = [_i, _vp, _i, _l, _vp, _i, _i, _i, _i, _i, _i, _vp, _vp, _vp, _i, _f, _vp, _l, _vp, _vp]
        K.ak_spec_verify.argtypes = [_vp, _l, _vp, _l, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp, _vp, _vp]
        _bound = K
    return _bound


# ------------------------------------------------------------------------------------------------ cache
def page_bytes(bits, page, heads, dim):
    n = heads * 2 * page * dim * bits // 8 + (heads * page * 4 if bits < 16 else 0)
    return (n + 127) // 128 * 128


def bf16_rn(x):
    """float64 -> bf16 bits, to nearest even from the 64-bit value (ties seen before any rounding to 32 bits)."""
    x = np.asarray(x, dtype=np.float64)
    _, e = np.frexp(np.where(np.isfinite(x), x, 0.0))
    ulp = np.ldexp(1.0, np.maximum(e - 8, -133))
    with np.errstate(invalid="ignore"):
        r = np.where(np.isfinite(x), np.round(x / ulp) * ulp, x)
    return f2bf_array(r.astype(np.float32)) if np.isfinite(r).all() else \
        np.where(np.isnan(r), 0x7FC0, f2bf_array(np.where(np.isnan(r), 0, r).astype(np.float32))).astype(np.uint16)


def quantise(x_bits, bits):
    """bf16 bits [..., dim] -> (codes as stored, scale bits [...]) by the definition, in 64 bits."""
    x = bf2f_array(x_bits).astype(np.float64)
    top, off = (127, 128) if bits == 8 else (7, 8)
    bad = ~np.isfinite(x).all(-1)
    amax = np.abs(np.where(np.isfinite(x), x, 0)).max(-1)
    s = bf16_rn(amax / top)
    s = np.where(s < 0x80, 0, s).astype(np.uint16)
    sv = bf2f_array(s).astype(np.float64)
    q = np.clip(np.round(x_safe(x) / np.where(sv > 0, sv, 1)[..., None]), -top, top) * (sv > 0)[..., None]
    q = np.where(bad[..., None], 0, q)
    return (q + off).astype(np.uint8), np.where(bad, 0x7FC0, s).astype(np.uint16)


def x_safe(x):
    return np.where(np.isfinite(x), x, 0.0)


def held(x_bits, bits):
    """The values that the cache holds of rows x, 64 bits."""
    if bits == 16:
        return bf2f_array(x_bits).astype(np.float64)
    c, s = quantise(x_bits, bits)
    return (c.astype(np.float64) - (128 if bits == 8 else 8)) * bf2f_array(s).astype(np.float64)[..., None]


class Pool:
    """A host image of the pages and its place on the device."""

    def __init__(self, bits, page, heads, dim, npages, fill=0xFF):
        self.bits, self.page, self.heads, self.dim, self.npages = bits, page, heads, dim, npages
        self.mem = np.full((npages, page_bytes(bits, page, heads, dim)), fill, dtype=np.uint8)  # 0xFFFF: NaN

    def put(self, slots, k_bits, v_bits):
        """Rows k, v [tokens][heads][dim] of bf16 bits into slots, byte by byte of the documented layout."""
        rb = self.dim * self.bits // 8
        plane = self.page * rb
        for t, slot in enumerate(slots):
            p, o = divmod(int(slot), self.page)
            for part, x in ((0, k_bits[t]), (1, v_bits[t])):
                if self.bits == 16:
                    raw, s = x.view(np.uint8).reshape(self.heads, rb), None
                else:
                    c, s = quantise(x, self.bits)
                    raw = c if self.bits == 8 else (c[:, 0::2] | (c[:, 1::2] << 4))
                for h in range(self.heads):
                    at = (2 * h + part) * plane + o * rb
                    self.mem[p, at:at + rb] = raw[h]
                    if s is not None:
                        at = 2 * self.heads * plane + (h * self.page + o) * 4 + 2 * part
                        self.mem[p, at:at + 2] = s[h:h + 1].view(np.uint8)


# ------------------------------------------------------------------------------------------------ attention
def attention64(q_bits, seqs, heads, kv, dim, scale):
    """q [m][heads][dim] bf16 bits; seqs: (first token, tokens, keys, values, present) per sequence, keys and values the
    held ones [len][kv][dim].  Returns y, lse, and for the tolerances mag = sum p |v| / sum p and zerr = the largest
    sum |q k| times the scale of a row."""
    m = q_bits.shape[0]
    y, lse = np.zeros((m, heads, dim)), np.full((m, heads), -np.inf)
    mag, zabs = np.zeros((m, heads, dim)), np.zeros((m, heads))
    g = heads // kv
    q = bf2f_array(q_bits).astype(np.float64).reshape(m, heads, dim)
    for first, count, k, v, present in seqs:
        for t in range(count):
            n = len(k) - count + t + 1
            if n <= 0:
                continue
            use = np.flatnonzero(present[:n])
            if not len(use):
                continue
            for h in range(heads):
                kk, vv = k[use, h // g], v[use, h // g]
                z = kk @ q[first + t, h] * scale
                top = z.max()
                e = np.exp(z - top)
                r = first + t
                y[r, h], lse[r, h] = e @ vv / e.sum(), top + np.log(e.sum())
                mag[r, h], zabs[r, h] = e @ np.abs(vv) / e.sum(), (np.abs(kk) @ np.abs(q[r, h])).max() * scale
    return y, lse, mag, zabs


# ------------------------------------------------------------------------------------------------ verification
def softmax64(l_bits, heat):
    """(probabilities, log probabilities, best) of bf16 logits, NaN as -inf; probabilities 0 where nothing is left."""
    l = bf2f_array(l_bits).astype(np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    top = l.max()
    if top == -np.inf:
        return np.zeros(len(l)), np.full(len(l), -np.inf), -1
    with np.errstate(invalid="ignore"):
        z = np.where(l == top, 0.0, (l - top) / heat)
    e = np.exp(z)
    return e / e.sum(), z - np.log(e.sum()), int(np.flatnonzero(l == top)[0])


def verify64(target, draft, ids, counts, u, temp, t):
    """One sequence.  target [t + 1][vocab] bits, draft [t][vocab] bits or None.  Returns tokens, accepted, logp and
    whether a decision lies so near its threshold (1e-5 of it) that 32-bit weights may take the other side."""
    n = min(max(counts, 0), t)
    greedy, heat = not temp > 0, (temp if temp > 0 else 1.0)
    tokens, logp, near = np.full(t + 1, -1, dtype=np.int32), np.zeros(t + 1), False
    for j in range(n + 1):
        p, lp, best = softmax64(target[j], heat)
        q = np.zeros_like(p)
        if j < n:
            x = int(ids[j])
            known = 0 <= x < len(p)
            if draft is not None:
                q = softmax64(draft[j], heat)[0]
            elif known:
                q[x] = 1.0
            if known:
                a, b = float(u[j]) * q[x], p[x]
                near |= (not greedy) and abs(a - b) <= 1e-5 * max(a, b) and max(a, b) > 0
                if (x == best) if greedy else a < b:
                    tokens[j], logp[j] = x, lp[x]
                    continue
        pick = best
        if not greedy and best >= 0:
            w = np.maximum(p - q, 0) if j < n else p
            if w.sum() <= 0:
                w = p
            near |= 0 < w.sum() < 1e-4  # what is left is rounding
            cdf = np.cumsum(w)
            at = float(u[t]) * cdf[-1]
            pick = int(np.flatnonzero(cdf > at)[0])
            gaps = cdf[pick] - at, at - (cdf[pick - 1] if pick else -1.0)
            near |= min(gaps) <= 1e-5 * cdf[-1]
        tokens[j] = pick
        logp[j] = lp[pick] if pick >= 0 else 0.0
        return tokens, j, logp, near


# ------------------------------------------------------------------------------------------------ streams and graphs
def hip():
    return ctypes.CDLL("libamdhip64.so")


class Stream:
    def __init__(self):
        ops()
        self.h = _vp()
        assert hip().hipStreamCreate(ctypes.byref(self.h)) == 0

    def sync(self):
        assert hip().hipStreamSynchronize(self.h) == 0

    def __del__(self):
        hip().hipStreamDestroy(self.h)


class Graph:
    """What `call(stream)` enqueues, captured."""

    def __init__(self, stream, call):
        self.graph, self.exe, self.stream = _vp(), _vp(), stream
        assert hip().hipStreamBeginCapture(stream.h, _i(1)) == 0  # thread-local capture mode
        rc = call(stream.h)
        assert hip().hipStreamEndCapture(stream.h, ctypes.byref(self.graph)) == 0
        assert rc == 0
        assert hip().hipGraphInstantiate(ctypes.byref(self.exe), self.graph, None, None, ctypes.c_size_t(0)) == 0

    def launch(self):
        assert hip().hipGraphLaunch(self.exe, self.stream.h) == 0

    def __del__(self):
        if self.exe:
            hip().hipGraphExecDestroy(self.exe)
        if self.graph:
            hip().hipGraphDestroy(self.graph)
