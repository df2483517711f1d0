"""Performance cases of the operators between the linears of a decode step: the paged key-value cache (quantised as it is
written, and read back), attention of new tokens over it, and the verification of drafted tokens.

`own` selects who computes: the C entry points of include/agens_kernels.h (ak_kv_write, ak_kv_read, ak_paged_attn,
ak_spec_verify) on torch's current stream, or the same operators in elementary torch operations.  Head counts and widths
are those of this repository's decoder (40 query heads and 8 key-value heads of 128, or one tensor-parallel rank's share of
them; 152064 logits) and generic ones around them.

Kinds of case:
  cache   the keys and values of m tokens written into pages of 16, 8 or 4 bits a value, and read back;
  attn    attention of t new tokens of each of b sequences over their pages, contexts of min_len to max_len tokens;
  verify  t drafted tokens of each of b sequences against the target's logits, from given uniform numbers.
"""
import ctypes
import importlib
import math

import torch

own = False

DEV = "cuda"
HEADS, KV_HEADS, DIM, VOCAB = 40, 8, 128, 152064
_vp, _i, _l, _f = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float
_lib = None


def lib():
    global _lib
    if _lib is None:
        k = importlib.import_module("agens-engine_amd").load()
        k.ak_kv_write.argtypes = [_i, _vp, _vp, _i, _l, _l, _vp, _vp, _i, _i, _i, _i, _vp]
        k.ak_kv_read.argtypes = [_i, _vp, _i, _i, _i, _i, _vp, _i, _vp, _vp, _l, _l, _vp]
        k.ak_paged_attn.argtypes = [_i, _vp, _i, _l, _vp, _i, _i, _i, _i, _i, _i, _vp, _vp, _vp, _i, _f, _vp, _l, _vp, _vp]
        k.ak_spec_verify.argtypes = [_vp, _l, _vp, _l, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp, _vp, _vp]
        _lib = k
    return _lib


def check(rc):
    if rc:
        raise RuntimeError("libagens_kernels: error %d" % rc)


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the new token of one conversation: the smallest call, bound by latency
        dict(name="cache_8bit_m1", kind="cache", bits=8, m=1, heads=KV_HEADS, dim=DIM, page=16),
        # a short prompt of odd length into 4 bits
        dict(name="cache_4bit_m333", kind="cache", bits=4, m=333, heads=KV_HEADS, dim=DIM, page=32),
        # a long prompt
        dict(name="cache_8bit_m16384", kind="cache", bits=8, m=16384, heads=KV_HEADS, dim=DIM, page=64),
        # one conversation with a short context
        dict(name="attn_8bit_b1_l777", kind="attn", bits=8, b=1, t=1, min_len=777, max_len=777, heads=HEADS,
             kv_heads=KV_HEADS, dim=DIM, page=16),
        # one conversation with a long context, nothing quantised: few rows, all the work along the cache
        dict(name="attn_16bit_b1_l131072", kind="attn", bits=16, b=1, t=1, min_len=131072, max_len=131072, heads=HEADS,
             kv_heads=KV_HEADS, dim=DIM, page=64),
        # a serving batch of unequal contexts
        dict(name="attn_8bit_b64_ragged", kind="attn", bits=8, b=64, t=1, min_len=129, max_len=16384, heads=HEADS,
             kv_heads=KV_HEADS, dim=DIM, page=32),
        # long contexts in 4 bits
        dict(name="attn_4bit_b16_l32768", kind="attn", bits=4, b=16, t=1, min_len=30001, max_len=32768, heads=HEADS,
             kv_heads=KV_HEADS, dim=DIM, page=64),
        # drafts of 8 tokens being verified for 4 conversations
        dict(name="attn_8bit_b4_t8_l8191", kind="attn", bits=8, b=4, t=8, min_len=4099, max_len=8191, heads=HEADS,
             kv_heads=KV_HEADS, dim=DIM, page=16),
        # one of eight tensor-parallel ranks: 5 query heads on one key-value head
        dict(name="attn_16bit_rank_b12", kind="attn", bits=16, b=12, t=1, min_len=1501, max_len=6007, heads=HEADS // 8,
             kv_heads=KV_HEADS // 8, dim=DIM, page=16),
        # one conversation, 4 drafted tokens with the draft model's logits
        dict(name="verify_b1_t4", kind="verify", b=1, t=4, vocab=VOCAB, draft=True),
        # drafts looked up in the prompt (no draft distribution), half of the sequences greedy
        dict(name="verify_b32_t5_lookup", kind="verify", b=32, t=5, vocab=VOCAB, draft=False),
        # a serving batch with drafts of 7 tokens and an odd vocabulary
        dict(name="verify_b24_t7_odd", kind="verify", b=24, t=7, vocab=100277, draft=True),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["cache", "attn", "attn", "attn", "verify"])
    bits, dim = rng.choice([16, 8, 8, 4]), rng.choice([64, 128, 128, 256])
    kv, page = rng.choice([1, 2, 3, 4, 8, 8]), rng.choice([16, 16, 32, 64, 128])
    if kind == "cache":
        return dict(kind=kind, bits=bits, m=_log(rng, 1, 8192), heads=kv, dim=dim, page=page)
    if kind == "verify":
        b, t = _log(rng, 1, 32), rng.choice([0, 1, 2, 3, 4, 5, 7, 8])
        return dict(kind=kind, b=b, t=t, vocab=_log(rng, 8000, VOCAB), draft=t > 0 and rng.random() < 0.6)
    group, b = rng.choice([1, 2, 4, 5, 5, 8]), _log(rng, 1, 64)
    t = rng.choice([1, 1, 1, rng.randint(2, 8)])
    # what the caches hold together stays below the largest listed case's
    cap = 400e6 / (b * kv * dim * bits / 4) / (1 if t == 1 else 4)
    hi = _log(rng, 16, max(17, min(131072, cap)))
    lo = max(t, hi if rng.random() < 0.3 else _log(rng, 1, hi))
    return dict(kind=kind, bits=bits, b=b, t=t, min_len=lo, max_len=max(lo, hi), heads=kv * group, kv_heads=kv, dim=dim,
                page=page)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)


def _randn(g, *shape):
    return torch.randn(shape, device=DEV, generator=g)


def _page_bytes(bits, page, heads, dim):
    n = heads * page * (2 * dim * bits // 8 + (4 if bits < 16 else 0))
    return (n + 127) // 128 * 128


def _lens(case):
    """Context lengths of the sequences: spread over their logarithm, the order mixed."""
    b, lo, hi = case["b"], case["min_len"], case["max_len"]
    lens = [int(round(lo * (hi / lo) ** (i / max(1, b - 1)))) for i in range(b)]
    step = next(s for s in (7, 11, 13, 17) if b % s) if b > 2 else 1
    return [lens[(i * step) % b] for i in range(b)][::-1]


def _kv_values(g, heads, n, dim):
    """Keys or values [n][heads][dim]: normal, with a few larger channels of each head."""
    x = _randn(g, n, heads, dim)
    return x * torch.where(torch.rand((1, heads, dim), device=DEV, generator=g) < 0.03, 4.0, 1.0)


def _codes(x, bits):
    """(codes, scales) of rows x [..., dim] in 8 or 4 bits: the values q * s they stand for, q = rint(x / s)."""
    top = 127.0 if bits == 8 else 7.0
    s = (x.abs().amax(-1) / top).to(torch.bfloat16).float()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    q = torch.where(s[..., None] > 0, x / s[..., None], torch.zeros_like(x)).round().clamp(-top, top)
    return q, s


def _pack(q, bits):
    """Codes [..., dim] as bytes: q + 128, or nibbles q + 8 with the even one low."""
    if bits == 8:
        return (q + 128).to(torch.uint8)
    n = (q + 8).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4)


def _row_views(pool, bits, page, heads, dim):
    """(rows, scales) of a pool [pages][bytes]: rows [pages][heads][2][page][bytes of a row], scales [pages][heads][page][2]."""
    rb = dim * bits // 8
    n = heads * 2 * page * rb
    rows = pool[:, :n].view(-1, heads, 2, page, rb) if pool.shape[1] == n else pool[:, :n].unflatten(1, (heads, 2, page, rb))
    if bits == 16:
        return rows, None
    return rows, pool[:, n:n + heads * page * 4].unflatten(1, (heads, page, 4))


def _fill_pool(g, case, npages):
    """A pool whose every slot holds a token's keys and values."""
    bits, page, heads, dim = case["bits"], case["page"], case["kv_heads"], case["dim"]
    pool = torch.zeros((npages, _page_bytes(bits, page, heads, dim)), dtype=torch.uint8, device=DEV)
    rows, scales = _row_views(pool, bits, page, heads, dim)
    step = max(1, (64 << 20) // (page * heads * dim * 2))
    for p in range(0, npages, step):
        n = min(step, npages - p)
        x = torch.stack([_kv_values(g, heads, n * page, dim) for _ in range(2)], 2)  # [tokens][heads][2][dim]
        x = x.to(torch.bfloat16).view(n, page, heads, 2, dim).permute(0, 2, 3, 1, 4)
        if bits == 16:
            rows[p:p + n] = x.contiguous().view(torch.uint8)
            continue
        q, s = _codes(x.float(), bits)
        rows[p:p + n] = _pack(q, bits)
        scales[p:p + n] = s.to(torch.bfloat16).permute(0, 1, 3, 2).contiguous().view(torch.uint8)
    return pool


def _prepare_cache(case, g):
    m, heads, dim, page = case["m"], case["heads"], case["dim"], case["page"]
    npages = (m + page - 1) // page + 3
    kv = [_kv_values(g, heads, m, dim).to(torch.bfloat16) for _ in range(2)]
    pages = torch.randperm(npages, device=DEV, generator=g)
    tok = torch.arange(m, device=DEV)
    slots = (pages[tok // page] * page + tok % page).to(torch.int32)
    pool = torch.zeros((npages, _page_bytes(case["bits"], page, heads, dim)), dtype=torch.uint8, device=DEV)
    return {"case": case, "k": kv[0], "v": kv[1], "slots": slots, "pool": pool, "npages": npages,
            "k_out": torch.empty_like(kv[0]), "v_out": torch.empty_like(kv[1])}


def _prepare_attn(case, g):
    lens, page, m = _lens(case), case["page"], case["b"] * case["t"]
    held = [(n + page - 1) // page for n in lens]
    npages = sum(held) + 5
    q = (_randn(g, m, case["heads"], case["dim"]) * 2.0).to(torch.bfloat16)
    order = torch.randperm(npages, device=DEV, generator=g).to(torch.int32)
    table = torch.full((case["b"], max(held) + 2), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    return {"case": case, "q": q, "pool": _fill_pool(g, case, npages), "npages": npages, "table": table, "lens_host": lens,
            "lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "scale": case["dim"] ** -0.5,
            "y": torch.empty_like(q), "lse": torch.empty((m, case["heads"]), dtype=torch.float32, device=DEV)}


def _prepare_verify(case, g):
    b, t, vocab = case["b"], case["t"], case["vocab"]
    target = _randn(g, b, t + 1, vocab) * 2.0
    # as trained models' logits: some tokens well above the rest
    likely = torch.randint(0, vocab, (b, t + 1, 48), device=DEV, generator=g)
    target.scatter_add_(2, likely, 16 + 8 * torch.rand(likely.shape, device=DEV, generator=g))
    temp = torch.rand((b,), device=DEV, generator=g) * 0.4 + 0.6
    if not case["draft"]:
        temp[::2] = 0.0  # greedy
    near = target[:, :t] + 0.3 * _randn(g, b, t, vocab)
    target, near = target.to(torch.bfloat16), near.to(torch.bfloat16)
    # drafted tokens: drawn from the draft's distribution
    noise = -torch.log(-torch.log(torch.rand((b, t, vocab), device=DEV, generator=g).clamp_(1e-20, 1 - 1e-7)))
    ids = (near.float() / temp.clamp(min=0.05)[:, None, None] + noise).argmax(-1).to(torch.int32) if t else \
        torch.zeros((b, 0), dtype=torch.int32, device=DEV)
    counts = torch.full((b,), t, dtype=torch.int32, device=DEV)
    if b > 2 and t > 1:
        counts[1::3] = t - 1  # some drafts are shorter
    u = torch.rand((b, t + 1), device=DEV, generator=g)
    return {"case": case, "target": target, "draft": near if case["draft"] else None, "ids": ids, "counts": counts, "u": u,
            "temp": temp, "tokens": torch.empty((b, t + 1), dtype=torch.int32, device=DEV),
            "accepted": torch.empty((b,), dtype=torch.int32, device=DEV),
            "logp": torch.empty((b, t + 1), dtype=torch.float32, device=DEV)}


def prepare(case, seed):
    g = _gen(seed)
    return {"cache": _prepare_cache, "attn": _prepare_attn, "verify": _prepare_verify}[case["kind"]](case, g)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    c, L, stream = s["case"], lib(), torch.cuda.current_stream().cuda_stream
    if c["kind"] == "cache":
        m, h, d = c["m"], c["heads"], c["dim"]
        check(L.ak_kv_write(c["bits"], s["k"].data_ptr(), s["v"].data_ptr(), m, h * d, h * d, s["slots"].data_ptr(),
                            s["pool"].data_ptr(), s["npages"], c["page"], h, d, stream))
        check(L.ak_kv_read(c["bits"], s["pool"].data_ptr(), s["npages"], c["page"], h, d, s["slots"].data_ptr(), m,
                           s["k_out"].data_ptr(), s["v_out"].data_ptr(), h * d, h * d, stream))
        return {"k": s["k_out"], "v": s["v_out"]}
    if c["kind"] == "attn":
        h, d = c["heads"], c["dim"]
        check(L.ak_paged_attn(c["bits"], s["q"].data_ptr(), s["q"].shape[0], h * d, s["pool"].data_ptr(), s["npages"],
                              c["page"], h, c["kv_heads"], d, c["b"], None, s["lens"].data_ptr(), s["table"].data_ptr(),
                              s["table"].shape[1], s["scale"], s["y"].data_ptr(), h * d, s["lse"].data_ptr(), stream))
        return {"y": s["y"], "lse": s["lse"]}
    v = c["vocab"]
    check(L.ak_spec_verify(s["target"].data_ptr(), v, s["draft"].data_ptr() if c["draft"] else None, v,
                           s["ids"].data_ptr(), s["counts"].data_ptr(), s["u"].data_ptr(), s["temp"].data_ptr(), c["b"],
                           c["t"], v, s["tokens"].data_ptr(), s["accepted"].data_ptr(), s["logp"].data_ptr(), stream))
    return {"tokens": s["tokens"], "accepted": s["accepted"], "logp": s["logp"]}


# ------------------------------------------------------------------------------------------------ the plain forms, 32 bits
def _plain_cache(s):
    c = s["case"]
    bits, page, heads, dim = c["bits"], c["page"], c["heads"], c["dim"]
    rows, scales = _row_views(s["pool"], bits, page, heads, dim)
    at, off = s["slots"].long() // page, s["slots"].long() % page
    x = torch.stack([s["k"], s["v"]], 2)  # [m][heads][2][dim]
    if bits == 16:
        rows.permute(0, 3, 1, 2, 4)[at, off] = x.contiguous().view(torch.uint8)
        back = rows.permute(0, 3, 1, 2, 4)[at, off].contiguous().view(torch.bfloat16)
        return {"k": back[:, :, 0], "v": back[:, :, 1]}
    q, sc = _codes(x.float(), bits)
    rows.permute(0, 3, 1, 2, 4)[at, off] = _pack(q, bits)
    scales.permute(0, 2, 1, 3)[at, off] = sc.to(torch.bfloat16).view(torch.uint8)
    q = _unpack(rows.permute(0, 3, 1, 2, 4)[at, off], bits)
    sc = scales.permute(0, 2, 1, 3)[at, off].contiguous().view(torch.bfloat16).float()
    back = (q * sc[..., None]).to(torch.bfloat16)
    return {"k": back[:, :, 0], "v": back[:, :, 1]}


def _unpack(b, bits):
    if bits == 8:
        return b.float() - 128
    return torch.stack([b & 15, b >> 4], -1).flatten(-2).float() - 8


def _plain_attn(s):
    c = s["case"]
    bits, page, kv, dim, t = c["bits"], c["page"], c["kv_heads"], c["dim"], c["t"]
    g = c["heads"] // kv
    rows, scales = _row_views(s["pool"], bits, page, kv, dim)
    y, lse = [], []
    for i, n in enumerate(s["lens_host"]):
        ids = s["table"][i, :(n + page - 1) // page].long()
        r = rows[ids]  # [pages][kv][2][page][bytes]
        if bits == 16:
            x = r.view(torch.bfloat16).float()
        else:
            sc = scales[ids].view(torch.bfloat16).float()  # [pages][kv][page][2]
            x = _unpack(r, bits) * sc.permute(0, 1, 3, 2)[..., None]
        x = x.permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n]  # [kv][2][tokens][dim]
        k, v = x[:, 0].contiguous(), x[:, 1].contiguous()
        q = s["q"][i * t:(i + 1) * t].float().view(t, kv, g, dim).permute(1, 0, 2, 3).reshape(kv, t * g, dim)
        z = torch.matmul(q, k.transpose(1, 2)) * s["scale"]  # [kv][t * g][tokens]
        seen = torch.arange(n, device=DEV)[None, :] < (n - t + 1 + torch.arange(t, device=DEV))[:, None]
        z = z.view(kv, t, g, n).masked_fill(~seen[None, :, None], -math.inf).view(kv, t * g, n)
        top = z.amax(-1, keepdim=True)
        e = torch.exp(z - top)
        total = e.sum(-1, keepdim=True)
        o = torch.matmul(e, v) / total
        y.append(o.view(kv, t, g, dim).permute(1, 0, 2, 3).reshape(t, kv * g, dim))
        lse.append((top + torch.log(total)).view(kv, t, g).permute(1, 0, 2).reshape(t, kv * g))
    return {"y": torch.cat(y).to(torch.bfloat16), "lse": torch.cat(lse)}


def _first(mask):
    """Index of the first true value along the last axis (its length where there is none)."""
    n = mask.shape[-1]
    at = torch.arange(n, device=mask.device)
    return torch.where(mask, at, n).amin(-1)


def _plain_verify(s):
    c = s["case"]
    b, t, vocab = c["b"], c["t"], c["vocab"]
    counts, ids, u, temp = s["counts"].long(), s["ids"].long(), s["u"], s["temp"]
    greedy = temp <= 0
    div = torch.where(greedy, torch.ones_like(temp), temp)[:, None, None]
    rows = torch.arange(b, device=DEV)
    z = s["target"].float()
    top = z.amax(-1, keepdim=True)
    best = _first(z == top)
    z = (z - top) / div
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    p = e / total
    logp = z - torch.log(total)
    px = p[:, :t].gather(2, ids[..., None])[..., 0]
    if c["draft"]:
        zq = s["draft"].float()
        eq = torch.exp((zq - zq.amax(-1, keepdim=True)) / div)
        q = eq / eq.sum(-1, keepdim=True)
        qx = q.gather(2, ids[..., None])[..., 0]
    else:
        q = torch.zeros((b, t, vocab), device=DEV).scatter_(2, ids[..., None], 1.0)
        qx = torch.ones((b, t), device=DEV)
    ok = torch.where(greedy[:, None], ids == best[:, :t], u[:, :t] * qx < px)
    ok &= torch.arange(t, device=DEV)[None] < counts[:, None]
    n = _first(~ok) if t else torch.zeros((b,), dtype=torch.long, device=DEV)
    w = p[rows, n]
    if t:
        rest = (w - q[rows, n.clamp(max=t - 1)]).clamp(min=0)
        rejected = (n < counts)[:, None] & (rest.sum(-1, keepdim=True) > 0)
        w = torch.where(rejected, rest, w)
    cdf = torch.cumsum(w, -1)
    pick = _first(cdf > u[:, t:t + 1] * cdf[:, -1:])
    pick = torch.where(greedy, best[rows, n], pick)
    place = torch.arange(t + 1, device=DEV)[None]
    tokens = torch.cat([ids, torch.zeros((b, 1), dtype=torch.long, device=DEV)], 1)
    tokens = torch.where(place < n[:, None], tokens, torch.where(place == n[:, None], pick[:, None], -1))
    lp = logp.gather(2, tokens.clamp(min=0)[..., None])[..., 0]
    return {"tokens": tokens.to(torch.int32), "accepted": n.to(torch.int32),
            "logp": torch.where(tokens >= 0, lp, torch.zeros_like(lp))}


def run(state):
    if own:
        return _own(state)
    return {"cache": _plain_cache, "attn": _plain_attn, "verify": _plain_verify}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------ what it takes
def work(case):
    kind = case["kind"]
    if kind == "cache":
        n = case["m"] * case["heads"] * case["dim"] * 2  # values; held once, written and read back
        held = n * case["bits"] / 8 + (case["m"] * case["heads"] * 4 if case["bits"] < 16 else 0)
        return {"bytes": n * 4 + 2 * held + 4 * case["m"], "flops": 8.0 * n}
    if kind == "attn":
        lens, t, dim = _lens(case), case["t"], case["dim"]
        token = case["kv_heads"] * (2 * dim * case["bits"] / 8 + (4 if case["bits"] < 16 else 0))
        pairs = sum(n * t - t * (t - 1) // 2 for n in lens)
        m = case["b"] * t
        return {"bytes": sum(lens) * token + m * case["heads"] * (4 * dim + 4) + 4 * sum(lens) / case["page"],
                "flops": 4.0 * pairs * case["heads"] * dim}
    rows = case["b"] * ((case["t"] + 1) + (case["t"] if case["draft"] else 0))
    return {"bytes": 2.0 * rows * case["vocab"], "flops": 6.0 * rows * case["vocab"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_row(x, bits):
    """What 8 or 4 bits hold of rows x [..., dim]: q * s in 64 bits, s a bfloat16."""
    if bits == 16:
        return x.double()
    top = 127 if bits == 8 else 7
    s = (x.double().abs().max(dim=-1, keepdim=True).values / top).bfloat16().double()
    return torch.where(s >= 2.0 ** -126, (x.double() / s).round().clamp(-top, top) * s, 0.0)


def _exact_cache(s):
    return {"k": _exact_row(s["k"], s["case"]["bits"]), "v": _exact_row(s["v"], s["case"]["bits"])}


def _exact_attn(s):
    c = s["case"]
    bits, page, kv, dim, t, heads = c["bits"], c["page"], c["kv_heads"], c["dim"], c["t"], c["heads"]
    rb, plane = dim * bits // 8, page * dim * bits // 8
    y = torch.zeros((c["b"] * t, heads, dim), dtype=torch.float64, device=DEV)
    lse = torch.zeros((c["b"] * t, heads), dtype=torch.float64, device=DEV)
    for i, n in enumerate(s["lens_host"]):
        ids = s["table"][i, :(n + page - 1) // page].long()
        for h in range(kv):
            kv64 = []
            for part in range(2):
                at = (2 * h + part) * plane
                raw = s["pool"][ids, at:at + plane].reshape(-1, rb)[:n].contiguous()
                if bits == 16:
                    kv64.append(raw.view(torch.bfloat16).double())
                    continue
                if bits == 8:
                    code = raw.double() - 128
                else:
                    code = torch.empty((n, dim), dtype=torch.float64, device=DEV)
                    code[:, 0::2], code[:, 1::2] = (raw % 16).double() - 8, (raw // 16).double() - 8
                at = 2 * kv * plane + h * page * 4
                sc = s["pool"][ids, at:at + 4 * page].reshape(-1, 4)[:n].contiguous().view(torch.bfloat16)[:, part]
                kv64.append(code * sc.double()[:, None])
            for j in range(t):
                seen = n - t + 1 + j
                for a in range(h * heads // kv, (h + 1) * heads // kv):
                    r = i * t + j
                    z = (kv64[0][:seen] @ s["q"][r, a].double()) * s["scale"]
                    lse[r, a] = torch.logsumexp(z, 0)
                    y[r, a] = torch.softmax(z, 0) @ kv64[1][:seen]
    return {"y": y, "lse": lse}


def _exact_verify(s):
    c = s["case"]
    b, t = c["b"], c["t"]
    tokens = torch.full((b, t + 1), -1, dtype=torch.int64)
    logp = torch.zeros((b, t + 1), dtype=torch.float64)
    accepted = torch.zeros((b,), dtype=torch.int64)
    ids, counts, u, temp = s["ids"].cpu(), s["counts"].cpu(), s["u"].double().cpu(), s["temp"].double().cpu()
    for i in range(b):
        heat = float(temp[i]) if temp[i] > 0 else 1.0
        n = 0
        while True:
            lp = torch.log_softmax(s["target"][i, n].double() / heat, 0)
            best = int((s["target"][i, n] == s["target"][i, n].max()).nonzero()[0, 0])
            drafted = n < int(counts[i])
            x = int(ids[i, n]) if drafted else best
            p = lp.exp()
            if drafted:
                q = torch.zeros_like(p)
                if c["draft"]:
                    q = torch.softmax(s["draft"][i, n].double() / heat, 0)
                else:
                    q[x] = 1.0
            if drafted and (x == best if temp[i] <= 0 else float(u[i, n] * q[x]) < float(p[x])):
                tokens[i, n], logp[i, n] = x, lp[x]
                n += 1
                continue
            if temp[i] > 0:
                w = p
                if drafted and float((p - q).clamp(min=0).sum()) > 0:
                    w = (p - q).clamp(min=0)
                cdf = w.cumsum(0)
                best = int((cdf > u[i, t].to(DEV) * cdf[-1]).nonzero()[0, 0])
            tokens[i, n], logp[i, n] = best, lp[best]
            break
        accepted[i] = n
    return {"tokens": tokens.int().to(DEV), "accepted": accepted.int().to(DEV), "logp": logp.to(DEV)}


def exact(case, seed):
    return {"cache": _exact_cache, "attn": _exact_attn, "verify": _exact_verify}[case["kind"]](prepare(case, seed))
