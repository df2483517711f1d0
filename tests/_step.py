"""Bindings and 64-bit restatements (numpy) of the operators of a batched step: pages and slots, rotary positions, sampling,
low-rank adapters.  Test infrastructure: the oracle."""
import ctypes
import math

import numpy as np

from _lib import check, Dev, bf2f_array, c_void_p, ptr_array, int_array
from _ops import ops, softmax64

_i, _l, _vp, _f, _d = ctypes.c_int, ctypes.c_long, c_void_p, ctypes.c_float, ctypes.c_double
_bound = None


def step():
    global _bound
    if _bound is None:
        K = ops()
        K.ak_kv_plan.argtypes = [_i, _i] + [_vp] * 6 + [_i, _i, _vp, _i] + [_vp] * 8
        K.ak_rope_freqs.argtypes = [_d, _i, _i, _d, _l, _d, _d, _vp, _vp]
        K.ak_rope.argtypes = [_vp, _l, _vp, _l, _i, _i, _i, _vp, _vp, _i, _i, _f, _vp]
        K.ak_rope_kv_write.argtypes = [_i, _vp, _l, _vp, _l, _vp, _l, _vp, _l, _i, _i, _vp, _vp, _i, _i, _f, _vp, _vp] + \
            [_i] * 4 + [_vp]
        K.ak_sample.argtypes = [_vp, _l, _vp, _vp, _vp, _vp, _vp, _i, _i, _vp, _vp, _vp]
        K.ak_lora_plan_bytes.argtypes, K.ak_lora_plan_bytes.restype = [_i, _i, _i, _i], ctypes.c_size_t
        K.ak_lora_plan.argtypes = [_vp, _i, _i, _vp, _vp]
        K.ak_lora_add.argtypes = [_vp, _vp, _i, _l, _i, _i, _i, _vp, _vp, _i] + [_vp] * 5 + [_vp]
        _bound = K
    return _bound


def i32(x):
    return np.asarray(x, dtype=np.int32)


# ------------------------------------------------------------------------------------------------ pages
def plan64(counts, drop, cached, held, table, free, nfree, page, npages, m, alloc=True):
    """The definition, a sequence and a token after another.  Returns what ak_kv_plan leaves, as a dict."""
    b, ldt = table.shape
    counts = [max(int(c), 0) for c in counts]
    cached = [max(int(c), 0) for c in cached]
    held = [min(max(int(h), 0), ldt) for h in held] if alloc else [0] * b
    table, free = table.copy(), free.copy()
    stack = min(max(int(nfree), 0), npages) if alloc else 0
    for i in range(b):
        if drop is not None and drop[i]:
            for j in range(held[i]):
                if stack < npages:
                    free[stack] = table[i, j]
                stack += 1
            cached[i] = held[i] = 0
    stack = min(stack, npages)
    out = {k: np.full(n, -1, dtype=np.int32) for k, n in (("pos", m), ("slots", m))}
    lens, refused, qstart, short = [], [], [0], False
    for i in range(b):
        qstart.append(qstart[-1] + counts[i])
        no = cached[i] + counts[i] > ldt * page or qstart[-1] > m
        need = -(-(cached[i] + counts[i]) // page) - held[i] if alloc else 0
        if not no and need > 0:
            short = short or need > stack
            no = short
        refused.append(int(no))
        lens.append(cached[i] + (0 if no else counts[i]))
        if no:
            continue
        for _ in range(max(need, 0)):
            stack -= 1
            table[i, held[i]] = free[stack]
            held[i] += 1
        for j in range(counts[i]):
            p = cached[i] + j
            out["pos"][qstart[i] + j] = p
            pg = int(table[i, p // page])
            out["slots"][qstart[i] + j] = pg * page + p % page if 0 <= pg < npages else -1
    return dict(out, lens=i32(lens), held=i32(held), nfree=i32([stack]), qstart=i32([min(q, m) for q in qstart]),
                refused=i32(refused), table=table, free=free)


# ------------------------------------------------------------------------------------------------ rotary positions
def rope64(x_bits, pos, freqs, rot, interleaved, mag):
    """Rows x [m][heads][dim] of bf16 bits, rotated, in 64 bits from angles in the longest floats there are."""
    x = bf2f_array(x_bits).astype(np.float64).reshape(x_bits.shape).astype(np.longdouble)
    a = (np.asarray(pos, dtype=np.longdouble)[:, None] * np.asarray(freqs, dtype=np.float64).astype(np.longdouble))[:, None]
    c, s = np.cos(a) * np.longdouble(mag), np.sin(a) * np.longdouble(mag)
    y = x.copy()
    if interleaved:
        u, v = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = u * c - v * s, v * c + u * s
    else:
        u, v = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = u * c - v * s, v * c + u * s
    return y.astype(np.float64)


def freqs64(theta, rot, scaling=0, factor=1.0, trained=1, slow=1.0, fast=32.0):
    j = np.arange(rot // 2)
    if scaling == 2:
        theta = theta * factor ** (rot / (rot - 2))
    f = theta ** (-2.0 * j / rot)
    if scaling == 1:
        f = f / factor
    if scaling == 3:
        keep = np.clip((trained * f / (2 * math.pi) - slow) / (fast - slow), 0, 1)
        f = f * (keep + (1 - keep) / factor)
    return f, (0.1 * math.log(factor) + 1 if scaling == 3 else 1.0)


# ------------------------------------------------------------------------------------------------ sampling
def sample64(bits, temp, top_k, top_p, min_p, u, tol=1e-5):
    """One row.  Returns the token, its log p, and whether a decision lies within `tol` of its threshold."""
    greedy, heat = not temp > 0, (temp if temp > 0 else 1.0)
    p, lp, best = softmax64(bits, heat)
    if greedy or best < 0:
        return best, (lp[best] if best >= 0 else 0.0), False
    l = bf2f_array(bits).astype(np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    order, near = np.argsort(-l, kind="stable"), False
    if 0 < top_k < len(l):
        order = order[:top_k]
    if top_p < 1:
        upto = np.cumsum(p[order])
        goal = max(float(np.float32(top_p)), 0.0) * upto[-1]
        n = max(1, int((upto < goal).sum()) + 1)
        # a token more or less moves sums by its own weight: only one that counts can change a decision
        gap = min(abs(upto[min(n, len(order)) - 1] - goal), abs(goal - (upto[n - 2] if n > 1 else 0.0)))
        near |= goal > 0 and gap <= tol * upto[-1] and p[order[min(n, len(order)) - 1]] > tol * upto[-1]
        order = order[:n]
    if min_p > 0:
        least = min(float(np.float32(min_p)), 1.0) * p.max()
        near |= bool(((np.abs(p[order] - least) <= tol * least) & (p[order] < p.max())).any())
        order = order[p[order] >= least]
    w = np.zeros_like(p)
    w[order] = p[order]
    cdf = np.cumsum(w)
    at = float(np.float32(u)) * cdf[-1]
    pick = int(np.flatnonzero(cdf > at)[0])
    near |= min(cdf[pick] - at, at - cdf[pick - 1] if pick and cdf[pick - 1] > 0 else np.inf) <= tol * cdf[-1]
    return pick, lp[pick], near


# ------------------------------------------------------------------------------------------------ adapters
def lora64(x_bits, ids, a_bits, b_bits, scale, base_bits, rank):
    """y per segment in 64 bits, and for the tolerances the sums of magnitudes: sum |B| sum |x A| scale."""
    x = bf2f_array(x_bits).astype(np.float64).reshape(x_bits.shape)
    y = [bf2f_array(v).astype(np.float64).reshape(v.shape) for v in base_bits]
    mag = [np.zeros_like(v) for v in y]
    for a in range(len(a_bits)):
        at = np.flatnonzero(np.asarray(ids) == a)
        if not len(at):
            continue
        A = bf2f_array(a_bits[a]).astype(np.float64).reshape(a_bits[a].shape)
        s, sm = x[at] @ A.T, np.abs(x[at]) @ np.abs(A).T
        c = 1.0 if scale is None else float(np.float32(scale[a]))
        for j, b in enumerate(b_bits):
            B = bf2f_array(b[a]).astype(np.float64).reshape(b[a].shape)
            y[j][at] += c * (s[:, j * rank:(j + 1) * rank] @ B.T)
            mag[j][at] += abs(c) * (sm[:, j * rank:(j + 1) * rank] @ np.abs(B).T)
    return y, mag
