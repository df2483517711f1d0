"""Performance cases of the operators that a batched decode step has around its linears: the batch's pages, slots and
positions, rotary positions (alone, and on the way into the paged cache), sampling, and low-rank adapters beside a linear.

`own` selects who computes: the C entry points of include/agens_kernels.h (ak_kv_plan, ak_rope, ak_rope_kv_write, ak_sample,
ak_lora_plan, ak_lora_add) on torch's current stream, or the same operators in elementary torch operations.  Sizes are those
of this repository's decoder (hidden 5120, 27648 inner values, 40 query heads and 8 key-value heads of 128, 152064 logits) and
generic ones around them.

Kinds of case:
  plan     pages for the new tokens of b sequences off the free list, and the positions and slots of these tokens;
  rope     queries and keys of m tokens rotated by their positions;
  rope_kv  the same, with the keys going straight into pages of 16 or 8 bits beside the values, read back where quantised;
  sample   one token of each of b rows of logits after temperature, top-k, top-p and min-p, from given uniform numbers;
  lora     low-rank products of m tokens of several adapters added to a linear's outputs.
"""
import ctypes
import importlib
import math

import torch

own = False

DEV = "cuda"
HIDDEN, INTER, HEADS, KV_HEADS, DIM, VOCAB = 5120, 27648, 40, 8, 128, 152064
_vp, _i, _l, _f = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float
_lib = None


def lib():
    global _lib
    if _lib is None:
        k = importlib.import_module("agens-engine_amd").load()
        k.ak_kv_plan.argtypes = [_i, _i] + [_vp] * 6 + [_i, _i, _vp, _i] + [_vp] * 8
        k.ak_rope.argtypes = [_vp, _l, _vp, _l, _i, _i, _i, _vp, _vp, _i, _i, _f, _vp]
        k.ak_rope_kv_write.argtypes = [_i, _vp, _l, _vp, _l, _vp, _l, _vp, _l, _i, _i, _vp, _vp, _i, _i, _f, _vp, _vp] + \
            [_i] * 4 + [_vp]
        k.ak_kv_read.argtypes = [_i, _vp, _i, _i, _i, _i, _vp, _i, _vp, _vp, _l, _l, _vp]
        k.ak_sample.argtypes = [_vp, _l, _vp, _vp, _vp, _vp, _vp, _i, _i, _vp, _vp, _vp]
        k.ak_lora_plan_bytes.argtypes, k.ak_lora_plan_bytes.restype = [_i, _i, _i, _i], ctypes.c_size_t
        k.ak_lora_plan.argtypes = [_vp, _i, _i, _vp, _vp]
        k.ak_lora_add.argtypes = [_vp, _vp, _i, _l, _i, _i, _i, _vp, _vp, _i] + [_vp] * 5 + [_vp]
        _lib = k
    return _lib


def check(rc):
    if rc:
        raise RuntimeError("libagens_kernels: error %d" % rc)


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the next token of one conversation: the smallest call, bound by latency
        dict(name="plan_b1", kind="plan", b=1, lo=1, hi=1, room=4096, page=16, dropped=False),
        # a serving step: most sequences take one token, every seventh begins with a prompt, some have ended
        dict(name="plan_b200_prompts", kind="plan", b=200, lo=1, hi=1501, room=4096, page=16, dropped=True),
        # one new token: 40 query heads and 8 key heads side by side
        dict(name="rope_m1", kind="rope", m=1, heads=HEADS + KV_HEADS, dim=DIM, rot=DIM, interleaved=False, far=131072,
             scaling=0),
        # a long prompt, neighbouring values paired, half of each head, at far positions of a stretched context
        dict(name="rope_m8191_interleaved_part", kind="rope", m=8191, heads=HEADS + KV_HEADS, dim=DIM, rot=DIM // 2,
             interleaved=True, far=1000000, scaling=3),
        # a decode batch into a cache of 8 bits
        dict(name="rope_kv_8bit_m48", kind="rope_kv", bits=8, m=48, heads=HEADS, kv_heads=KV_HEADS, dim=DIM, rot=DIM, page=16,
             interleaved=False, far=32768, scaling=0),
        # a long prompt into a cache of 16 bits
        dict(name="rope_kv_16bit_m8192", kind="rope_kv", bits=16, m=8192, heads=HEADS, kv_heads=KV_HEADS, dim=DIM, rot=DIM,
             page=64, interleaved=False, far=8192, scaling=2),
        # one conversation's next token
        dict(name="sample_b1", kind="sample", b=1, vocab=VOCAB, peaks=48),
        # a serving batch whose requests each have settings of their own, some greedy, some without any filter
        dict(name="sample_b32_mixed", kind="sample", b=32, vocab=VOCAB, peaks=48),
        # a large batch, an odd vocabulary, flat rows: filters that keep tens of thousands of tokens
        dict(name="sample_b250_flat", kind="sample", b=250, vocab=100277, peaks=0),
        # one token of one adapter beside the output projection
        dict(name="lora_o_m1", kind="lora", m=1, adapters=4, used=1, rank=16, k=HIDDEN, n="%d" % HIDDEN),
        # a decode batch of many adapters beside the merged q, k and v
        dict(name="lora_qkv_m64", kind="lora", m=64, adapters=32, used=24, rank=16, k=HIDDEN,
             n="%d+%d+%d" % (HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM)),
        # prompts of three adapters beside the down projection
        dict(name="lora_down_m4001", kind="lora", m=4001, adapters=4, used=3, rank=64, k=INTER, n="%d" % HIDDEN),
    ]


def _rows(case):
    """Output rows of the segments that share x: "5120+1024+1024"."""
    return [int(v) for v in case["n"].split("+")]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["plan", "rope", "rope_kv", "sample", "sample", "lora", "lora"])
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "plan":
        return dict(kind=kind, b=_log(rng, 1, 512), lo=1, hi=_log(rng, 1, 1000), room=_log(rng, 2048, 16384), page=page,
                    dropped=rng.random() < 0.5)
    if kind in ("rope", "rope_kv"):
        dim = rng.choice([64, 128, 128, 256] if kind == "rope_kv" else [64, 80, 96, 128, 128, 256])
        kv, group = rng.choice([1, 2, 3, 4, 8, 8]), rng.choice([1, 2, 4, 5])
        rot = dim if rng.random() < 0.6 else 2 * rng.randint(4, dim // 2)
        c = dict(kind=kind, m=_log(rng, 1, min(8192, 8192 * 48 * 128 // (kv * (group + 2) * dim))), dim=dim, rot=rot,
                 interleaved=rng.random() < 0.4, far=_log(rng, 8192, 1000000), scaling=rng.choice([0, 0, 1, 2, 3]))
        if kind == "rope":
            return dict(c, heads=kv * (group + 1))
        return dict(c, bits=rng.choice([16, 8]), heads=kv * group, kv_heads=kv, page=page)
    if kind == "sample":
        vocab = _log(rng, 1000, VOCAB)
        return dict(kind=kind, b=_log(rng, 1, min(512, 25000000 // vocab)), vocab=vocab, peaks=rng.choice([0, 0, 1, 48, 48]))
    k = rng.choice([1024, 2048, 4096, HIDDEN, HIDDEN, INTER // 8, INTER])
    rank = rng.choice([8, 16, 16, 32, 64])
    n = [rng.choice([640, 1024, 2055, HIDDEN, 7168]) for _ in range(rng.choice([1, 1, 2, 3]))]
    adapters = _log(rng, 1, 64)
    m = _log(rng, 1, max(2, min(4000, 4000 * (INTER + HIDDEN) // (k + sum(n)) * 64 // (rank * len(n)))))
    return dict(kind=kind, m=m, adapters=adapters, used=rng.randint(1, adapters), rank=rank, k=k,
                n="+".join(map(str, n)))


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)


def _randn(g, *shape):
    return torch.randn(shape, device=DEV, generator=g)


def _int(*shape):
    return torch.zeros(shape, dtype=torch.int32, device=DEV)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _counts(case):
    """New tokens of each sequence: one each, a prompt for every seventh."""
    b, lo, hi = case["b"], case["lo"], case["hi"]
    return [lo if i % 7 != 3 or hi == lo else int(round(lo + (hi - lo) * (i + 1) / b)) for i in range(b)]


def _prepare_plan(case, g, seed):
    b, page, room = case["b"], case["page"], case["room"]
    ldt = (room + page - 1) // page
    counts = _counts(case)
    # contexts of any length up to the room, the order mixed
    cached = [min(room - c, int(room * (0.02 + 0.9 * (i * 37 + 11) % 97 / 97))) if c == case["lo"] else 0
              for i, c in enumerate(counts)]
    drop = [0] * b
    if case["dropped"]:
        for i in range(5, b, 11):  # ended: its pages go back, its row takes nothing yet
            drop[i], counts[i] = 1, 0
    held = [(n + page - 1) // page for n in cached]
    extra = sum(c // page + 2 for c in counts)
    npages = sum(held) + extra + 3
    order = torch.randperm(npages, device=DEV, generator=g).to(torch.int32)
    table = torch.full((b, ldt), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    free = torch.full((npages,), -1, dtype=torch.int32, device=DEV)
    free[:npages - at] = order[at:]
    m = sum(counts) + 5  # a captured step's rows, the last ones unused
    return {"case": case, "m": m, "ldt": ldt, "npages": npages, "counts": _i32(counts), "drop": _i32(drop),
            "cached": _i32(cached), "held": _i32(held), "nfree": _i32([npages - at]), "free": free, "table": table,
            "lens": _int(b), "held_out": _int(b), "nfree_out": _int(1), "qstart": _int(b + 1), "pos": _int(m),
            "slots": _int(m), "refused": _int(b)}


THETA, TRAINED = 1000000.0, 8192


def _freqs(case):
    """Radians per position of each pair (64 bits, on the host, as a program makes them when it loads a model), and the factor
    of the rotated values: plain, positions divided by 8, a larger base, or slow pairs divided by 8 and fast ones left."""
    rot, kind, factor = case["rot"], case["scaling"], 8.0
    theta = THETA * factor ** (rot / (rot - 2)) if kind == 2 else THETA
    f = [theta ** (-2.0 * j / rot) for j in range(rot // 2)]
    if kind == 1:
        f = [v / factor for v in f]
    if kind == 3:
        keep = [min(1.0, max(0.0, (TRAINED * v / (2 * math.pi) - 1.0) / (32.0 - 1.0))) for v in f]
        f = [v * (k + (1 - k) / factor) for v, k in zip(f, keep)]
    return torch.tensor(f, dtype=torch.float64), (0.1 * math.log(factor) + 1 if kind == 3 else 1.0)


def _positions(case, g):
    """Tokens of up to eight sequences side by side, each from a position of its own on."""
    m = case["m"]
    each = (m + 7) // 8
    first = (torch.rand((8,), device=DEV, generator=g) * max(1, case["far"] - each)).long()
    t = torch.arange(m, device=DEV)
    return (first[t // each] + t % each).to(torch.int32)


def _heads(g, m, heads, dim):
    """Queries, keys or values [m][heads][dim]: normal, with a few larger channels of each head."""
    return _randn(g, m, heads, dim) * torch.where(torch.rand((1, heads, dim), device=DEV, generator=g) < 0.03, 4.0, 1.0)


def _prepare_rope(case, g, seed):
    x = _heads(g, case["m"], case["heads"], case["dim"]).to(torch.bfloat16)
    f, mag = _freqs(case)
    return {"case": case, "x": x, "pos": _positions(case, g), "freqs": f.to(DEV), "mag": mag, "y": torch.empty_like(x)}


def _page_bytes(bits, page, heads, dim):
    n = heads * page * (2 * dim * bits // 8 + (4 if bits < 16 else 0))
    return (n + 127) // 128 * 128


def _prepare_rope_kv(case, g, seed):
    m, kv, dim, page = case["m"], case["kv_heads"], case["dim"], case["page"]
    qkv = _heads(g, m, case["heads"] + 2 * kv, dim).to(torch.bfloat16)  # a merged projection's output
    f, mag = _freqs(case)
    npages = (m + page - 1) // page + 3
    tok = torch.arange(m, device=DEV)
    slots = torch.randperm(npages, device=DEV, generator=g)[tok // page] * page + tok % page
    pool = torch.zeros((npages, _page_bytes(case["bits"], page, kv, dim)), dtype=torch.uint8, device=DEV)
    kv_out = [torch.empty((m, kv, dim), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    return {"case": case, "qkv": qkv, "pos": _positions(case, g), "freqs": f.to(DEV), "mag": mag, "slots": slots.to(torch.int32),
            "pool": pool, "npages": npages, "q": torch.empty((m, case["heads"], dim), dtype=torch.bfloat16, device=DEV),
            "k_out": kv_out[0], "v_out": kv_out[1]}


def _prepare_sample(case, g, seed):
    b, vocab = case["b"], case["vocab"]
    z = _randn(g, b, vocab) * (2.0 if case["peaks"] else 1.5)
    if case["peaks"]:  # as trained models' logits: some tokens well above the rest
        likely = torch.randint(0, vocab, (b, case["peaks"]), device=DEV, generator=g)
        z.scatter_add_(1, likely, 16 + 8 * torch.rand(likely.shape, device=DEV, generator=g))
    r = torch.rand((b, 8), device=DEV, generator=g)
    temp = 0.3 + 1.2 * r[:, 0]
    top_k = torch.where(r[:, 1] < 0.5, 0, torch.exp(r[:, 2] * math.log(min(vocab, 2000))).int() + 1).to(torch.int32)
    top_p = torch.where(r[:, 3] < 0.3, 1.0, 0.5 + 0.49 * r[:, 4])
    min_p = torch.where(r[:, 5] < 0.6, 0.0, 0.001 + 0.1 * r[:, 6])
    if b > 2:
        temp[::8] = 0.0  # greedy
        top_k[1::8], top_p[1::8], min_p[1::8] = 0, 1.0, 0.0  # no filter
    return {"case": case, "logits": z.to(torch.bfloat16), "temp": temp, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "u": r[:, 7].contiguous(), "tokens": _int(b), "logp": torch.empty((b,), device=DEV)}


def _prepare_lora(case, g, seed):
    m, k, r, n, ad = case["m"], case["k"], case["rank"], _rows(case), case["adapters"]
    host = torch.Generator().manual_seed(int(seed) & 0x7FFFFFFF)
    names = torch.randperm(ad, generator=host)[:case["used"]]
    if m <= 256:  # a decode batch: every token is another request's
        ids = names[torch.randint(0, case["used"], (m,), generator=host)]
        if m > 8:
            ids[3::9] = -1  # requests without an adapter
    else:  # prompts of up to eight requests side by side
        ids = names[torch.arange(8) % case["used"]][torch.arange(m) * 8 // m].clone()
        ids[m - m // 8:] = -1
    a = torch.cat([_randn(g, 1, len(n) * r, k) * k ** -0.5 for _ in range(ad)]).to(torch.bfloat16)
    bs = [(_randn(g, ad, ni, r) * (0.5 * r ** -0.5)).to(torch.bfloat16) for ni in n]
    x = _randn(g, m, k).to(torch.bfloat16)
    y0 = [_randn(g, m, ni).to(torch.bfloat16) for ni in n]
    s = {"case": case, "ids_host": ids.tolist(), "ids": ids.to(torch.int32).to(DEV), "x": x, "a": a, "b": bs, "y0": y0,
         "scale": torch.linspace(0.5, 2.0, ad, device=DEV), "y": [torch.empty_like(t) for t in y0]}
    if own:
        s["plan"] = torch.zeros(lib().ak_lora_plan_bytes(m, ad, len(n) * r, k), dtype=torch.uint8, device=DEV)
    return s


def prepare(case, seed):
    kinds = {"plan": _prepare_plan, "rope": _prepare_rope, "rope_kv": _prepare_rope_kv, "sample": _prepare_sample,
             "lora": _prepare_lora}
    return kinds[case["kind"]](case, _gen(seed), seed)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _p(t):
    return t.data_ptr()


def _ptrs(ts):
    return (_vp * len(ts))(*[t.data_ptr() for t in ts])


def _own(s):
    c, L, stream = s["case"], lib(), torch.cuda.current_stream().cuda_stream
    kind = c["kind"]
    if kind == "plan":
        check(L.ak_kv_plan(c["b"], s["m"], _p(s["counts"]), _p(s["drop"]), _p(s["cached"]), _p(s["held"]), _p(s["nfree"]),
                           _p(s["free"]), s["npages"], c["page"], _p(s["table"]), s["ldt"], _p(s["lens"]), _p(s["held_out"]),
                           _p(s["nfree_out"]), _p(s["qstart"]), _p(s["pos"]), _p(s["slots"]), _p(s["refused"]), stream))
        return {"lens": s["lens"], "held": s["held_out"], "nfree": s["nfree_out"], "qstart": s["qstart"], "pos": s["pos"],
                "slots": s["slots"], "refused": s["refused"], "table": s["table"], "free": s["free"]}
    if kind == "rope":
        w = c["heads"] * c["dim"]
        check(L.ak_rope(_p(s["x"]), w, _p(s["y"]), w, c["m"], c["heads"], c["dim"], _p(s["pos"]), _p(s["freqs"]), c["rot"],
                        int(c["interleaved"]), s["mag"], stream))
        return {"y": s["y"]}
    if kind == "rope_kv":
        h, kv, d, m, page = c["heads"], c["kv_heads"], c["dim"], c["m"], c["page"]
        w = (h + 2 * kv) * d
        check(L.ak_rope_kv_write(c["bits"], _p(s["qkv"]), w, _p(s["qkv"]) + 2 * h * d, w, _p(s["qkv"]) + 2 * (h + kv) * d, w,
                                 _p(s["q"]), h * d, m, h, _p(s["pos"]), _p(s["freqs"]), c["rot"], int(c["interleaved"]),
                                 s["mag"], _p(s["slots"]), _p(s["pool"]), s["npages"], page, kv, d, stream))
        if c["bits"] == 16:
            return {"q": s["q"], "pool": s["pool"].view(torch.bfloat16)}
        check(L.ak_kv_read(c["bits"], _p(s["pool"]), s["npages"], page, kv, d, _p(s["slots"]), m, _p(s["k_out"]),
                           _p(s["v_out"]), kv * d, kv * d, stream))
        return {"q": s["q"], "k": s["k_out"], "v": s["v_out"]}
    if kind == "sample":
        check(L.ak_sample(_p(s["logits"]), c["vocab"], _p(s["temp"]), _p(s["top_k"]), _p(s["top_p"]), _p(s["min_p"]), _p(s["u"]),
                          c["b"], c["vocab"], _p(s["tokens"]), _p(s["logp"]), stream))
        return {"tokens": s["tokens"], "logp": s["logp"]}
    n = _rows(c)
    check(L.ak_lora_plan(_p(s["ids"]), c["m"], c["adapters"], _p(s["plan"]), stream))
    check(L.ak_lora_add(_p(s["plan"]), _p(s["x"]), c["m"], c["k"], c["k"], c["adapters"], c["rank"], _p(s["a"]), _p(s["scale"]),
                        len(n), _ptrs(s["b"]), _ptrs(s["y0"]), _ptrs(s["y"]), (_i * len(n))(*n), None, stream))
    return {"y%d" % j: y for j, y in enumerate(s["y"])}


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_plan(s):
    c, m, ldt, npages = s["case"], s["m"], s["ldt"], s["npages"]
    b, page = c["b"], c["page"]
    counts, gone = s["counts"].long().clamp(min=0), s["drop"] != 0
    zero = torch.zeros_like(counts)
    n, h = torch.where(gone, zero, s["cached"].long()), torch.where(gone, zero, s["held"].long())
    back = torch.where(gone, s["held"].long(), zero)
    col = torch.arange(ldt, device=DEV)[None]
    # pages of ended sequences onto the free list (what is not given back goes to a spare place behind it)
    free = torch.cat([s["free"], _int(1)])
    to = s["nfree"].long() + (torch.cumsum(back, 0) - back)[:, None] + col
    free.scatter_(0, torch.where(col < back[:, None], to, npages).flatten(), s["table"].flatten())
    avail = s["nfree"].long() + back.sum()
    # pages off its end
    qend = torch.cumsum(counts, 0)
    out = ((n + counts) > ldt * page) | (qend > m)
    want = torch.where(out, zero, ((n + counts + page - 1) // page - h).clamp(min=0))
    upto = torch.cumsum(want, 0)
    refused = out | ((want > 0) & (upto > avail))
    take = torch.where(refused, zero, want)
    place = avail - 1 - ((upto - want)[:, None] + col - h[:, None])
    new = (col >= h[:, None]) & (col < (h + take)[:, None])
    table = torch.where(new, free[place.clamp(0, npages)], s["table"])
    # the tokens
    t = torch.arange(m, device=DEV)
    seq = torch.searchsorted(qend, t, right=True).clamp(max=b - 1)
    p = n[seq] + t - (qend - counts)[seq]
    there = (t < qend[-1]) & ~refused[seq]
    p = torch.where(there, p, -1)
    pg = table[seq, p.clamp(min=0) // page].long()
    slots = torch.where(there & (pg >= 0) & (pg < npages), pg * page + p % page, -1)
    qstart = torch.cat([zero[:1], qend]).clamp(max=m)
    lens = torch.where(refused, n, n + counts)
    i = torch.int32
    return {"lens": lens.to(i), "held": (h + take).to(i), "nfree": (avail - take.sum()).to(i), "qstart": qstart.to(i),
            "pos": p.to(i), "slots": slots.to(i), "refused": refused.to(i), "table": table, "free": free[:npages]}


def _rotate(x, pos, freqs, c, mag, wide):
    """x [m][heads][dim] rotated; angles in 64 bits, products in 32 (64 where `wide`)."""
    rot = c["rot"]
    angle = pos.double()[:, None] * freqs[None]
    t = torch.float64 if wide else torch.float32
    cos, sin = (torch.cos(angle) * mag).to(t)[:, None], (torch.sin(angle) * mag).to(t)[:, None]
    x = x.to(t)
    if c["interleaved"]:
        u, v = x[..., 0:rot:2], x[..., 1:rot:2]
        r = torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
    else:
        u, v = x[..., :rot // 2], x[..., rot // 2:rot]
        r = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
    return torch.cat([r, x[..., rot:]], -1)


def _plain_rope(s):
    return {"y": _rotate(s["x"], s["pos"], s["freqs"], s["case"], s["mag"], False).to(torch.bfloat16)}


def _codes(x, top):
    """(codes, scales) of rows x [..., dim] as floats: the values q * s they stand for, q = rint(x / s)."""
    s = (x.abs().amax(-1) / top).to(torch.bfloat16).float()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    return torch.where(s[..., None] > 0, x / s[..., None], torch.zeros_like(x)).round().clamp(-top, top), s


def _near(x):
    """64 bits -> the nearest bfloat16 (a step over 32 bits would move values next to a border)."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -126))) - 7)
    return (torch.round(x / step) * step).to(torch.bfloat16)


def _plain_rope_kv(s):
    c = s["case"]
    bits, h, kv, dim, page = c["bits"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    q = _rotate(s["qkv"][:, :h], s["pos"], s["freqs"], c, s["mag"], False).to(torch.bfloat16)
    k = _near(_rotate(s["qkv"][:, h:h + kv], s["pos"], s["freqs"], c, s["mag"], True))
    x = torch.stack([k, s["qkv"][:, h + kv:]], 2)  # [m][kv][2][dim]
    rb = dim * bits // 8
    n = kv * 2 * page * rb
    rows = s["pool"][:, :n].unflatten(1, (kv, 2, page, rb)).permute(0, 3, 1, 2, 4)
    at, off = s["slots"].long() // page, s["slots"].long() % page
    if bits == 16:
        rows[at, off] = x.contiguous().view(torch.uint8)
        return {"q": q, "pool": s["pool"].view(torch.bfloat16)}
    code, sc = _codes(x.float(), 127.0)
    scales = s["pool"][:, n:n + kv * page * 4].unflatten(1, (kv, page, 4)).permute(0, 2, 1, 3)
    rows[at, off] = (code + 128).to(torch.uint8)
    scales[at, off] = sc.to(torch.bfloat16).view(torch.uint8)
    back = (rows[at, off].float() - 128) * scales[at, off].contiguous().view(torch.bfloat16).float()[..., None]
    back = back.to(torch.bfloat16)
    return {"q": q, "k": back[:, :, 0], "v": back[:, :, 1]}


def _first(mask):
    """Index of the first true value along the last axis (its length where there is none)."""
    n = mask.shape[-1]
    at = torch.arange(n, device=mask.device)
    return torch.where(mask, at, n).amin(-1)


def _plain_sample(s):
    vocab = s["case"]["vocab"]
    z = s["logits"].float()
    greedy = s["temp"] <= 0
    top = z.amax(-1, keepdim=True)
    best = _first(z == top)
    z = (z - top) / torch.where(greedy, 1.0, s["temp"])[:, None]
    e = torch.exp(z)
    logp = z - torch.log(e.sum(-1, keepdim=True))
    # by falling weight, the lower token first among equal ones
    w, order = torch.sort(e, dim=-1, descending=True, stable=True)
    rank = torch.arange(vocab, device=DEV)[None]
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    w = torch.where(rank < k, w, 0.0)
    upto = torch.cumsum(w, -1, dtype=torch.float64)  # (64 bits: long sums against a border)
    keep = (upto - w < s["top_p"].double()[:, None] * upto[:, -1:]) | (s["top_p"] >= 1)[:, None] | (rank == 0)
    keep &= (rank < k) & (w >= s["min_p"][:, None])
    kept = torch.zeros_like(e).scatter_(1, order, torch.where(keep, w, 0.0))
    cdf = torch.cumsum(kept, -1, dtype=torch.float64)
    pick = _first(cdf > s["u"].double()[:, None] * cdf[:, -1:])
    pick = torch.where(greedy, best, pick)
    return {"tokens": pick.to(torch.int32), "logp": logp.gather(1, pick[:, None])[:, 0]}


def _plain_lora(s):
    c, r = s["case"], s["case"]["rank"]
    out = [t.clone() for t in s["y0"]]
    for a in sorted(set(s["ids_host"]) - {-1}):
        at = torch.tensor([t for t, v in enumerate(s["ids_host"]) if v == a], device=DEV)
        down = s["x"][at].float() @ s["a"][a].float().t() * s["scale"][a]
        for j, y in enumerate(out):
            y[at] = (s["y0"][j][at].float() + down[:, j * r:(j + 1) * r] @ s["b"][j][a].float().t()).to(torch.bfloat16)
    return {"y%d" % j: y for j, y in enumerate(out)}


def run(state):
    if own:
        return _own(state)
    kinds = {"plan": _plain_plan, "rope": _plain_rope, "rope_kv": _plain_rope_kv, "sample": _plain_sample, "lora": _plain_lora}
    return kinds[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------ what it takes
def work(case):
    kind = case["kind"]
    if kind == "plan":
        counts = _counts(case)
        pages = sum((n + case["page"] - 1) // case["page"] for n in counts)
        return {"bytes": 4.0 * (9 * case["b"] + 3) + 8.0 * sum(counts) + 8.0 * pages, "flops": 4.0 * sum(counts)}
    if kind == "rope":
        n = case["m"] * case["heads"] * case["dim"]
        return {"bytes": 4.0 * n + 4 * case["m"], "flops": 3.0 * case["m"] * case["heads"] * case["rot"]}
    if kind == "rope_kv":
        m, d, kv, bits = case["m"], case["dim"], case["kv_heads"], case["bits"]
        held = m * kv * (2 * d * bits / 8 + (4 if bits < 16 else 0))
        back = held + 4.0 * m * kv * d if bits < 16 else 0.0
        return {"bytes": 4.0 * m * case["heads"] * d + 4.0 * m * kv * d + held + back + 8 * m,
                "flops": 3.0 * m * (case["heads"] + kv) * case["rot"]}
    if kind == "sample":
        return {"bytes": 2.0 * case["b"] * case["vocab"], "flops": 6.0 * case["b"] * case["vocab"]}
    m, k, r, n = case["m"], case["k"], case["rank"], _rows(case)
    used = min(case["used"], m)
    return {"bytes": 2.0 * m * k + 4.0 * m * sum(n) + 2.0 * used * r * (len(n) * k + sum(n)) + 4 * m,
            "flops": 2.0 * m * r * (len(n) * k + sum(n))}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_plan(s):
    """One sequence and one token after another, as the definition reads."""
    c, m, ldt, page, npages = s["case"], s["m"], s["ldt"], s["case"]["page"], s["npages"]
    b = c["b"]
    counts, drop, cached, held = (s[k].tolist() for k in ("counts", "drop", "cached", "held"))
    table, free, stack = s["table"].tolist(), s["free"].tolist(), s["nfree"].tolist()[0]
    for i in range(b):
        if drop[i]:
            for j in range(held[i]):
                free[stack] = table[i][j]
                stack += 1
            cached[i] = held[i] = 0
    qstart, lens, refused, short = [0], [], [], False
    pos, slots = [-1] * m, [-1] * m
    for i in range(b):
        qstart.append(qstart[-1] + counts[i])
        need = -(-(cached[i] + counts[i]) // page) - held[i]
        no = cached[i] + counts[i] > ldt * page or qstart[-1] > m
        if not no and need > 0:
            short = short or need > stack
            no = short
        refused.append(int(no))
        lens.append(cached[i] + (0 if no else counts[i]))
        if no:
            continue
        for _ in range(max(0, need)):
            stack -= 1
            table[i][held[i]] = free[stack]
            held[i] += 1
        for j in range(counts[i]):
            p = cached[i] + j
            pos[qstart[i] + j], slots[qstart[i] + j] = p, table[i][p // page] * page + p % page
    return {"lens": _i32(lens), "held": _i32(held), "nfree": _i32([stack]), "qstart": _i32([min(v, m) for v in qstart]),
            "pos": _i32(pos), "slots": _i32(slots), "refused": _i32(refused), "table": _i32(table), "free": _i32(free)}


def _exact_turn(x, s):
    """Rotation as a product of complex numbers."""
    c = s["case"]
    rot, m, heads = c["rot"], x.shape[0], x.shape[1]
    x = x.double()
    z = x[..., :rot].reshape(m, heads, rot // 2, 2) if c["interleaved"] else \
        x[..., :rot].reshape(m, heads, 2, rot // 2).transpose(2, 3)
    angle = s["pos"].double()[:, None, None] * s["freqs"]
    z = torch.view_as_complex(z.contiguous()) * torch.polar(torch.full_like(angle, s["mag"]), angle)
    z = torch.view_as_real(z)
    z = (z if c["interleaved"] else z.transpose(2, 3)).reshape(m, heads, rot)
    return torch.cat([z, x[..., rot:]], -1)


def _exact_rope(s):
    return {"y": _exact_turn(s["x"], s)}


def _exact_rope_kv(s):
    c = s["case"]
    m, h, kv, dim, page = c["m"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    q, k, v = _exact_turn(s["qkv"][:, :h], s), _exact_turn(s["qkv"][:, h:h + kv], s), s["qkv"][:, h + kv:].double()
    if c["bits"] == 16:
        out = torch.zeros((s["npages"], kv, 2, page, dim), dtype=torch.float64, device=DEV)
        for part, x in ((0, k), (1, v)):
            out[s["slots"].long() // page, :, part, s["slots"].long() % page] = x
        return {"q": q, "pool": out.flatten(1)}
    held = []
    for x in (k, v):  # the cache holds codes of the keys as bfloat16
        mant, e = torch.frexp(x)
        x = torch.ldexp(torch.round(mant * 256), e - 8)
        sc = (x.abs().amax(-1, keepdim=True) / 127).bfloat16().double()
        held.append(torch.where(sc >= 2.0 ** -126, (x / sc).round().clamp(-127, 127) * sc, 0.0))
    return {"q": q, "k": held[0], "v": held[1]}


def _exact_sample(s):
    c = s["case"]
    temp, top_k, top_p, min_p, u = (s[k].double().tolist() for k in ("temp", "top_k", "top_p", "min_p", "u"))
    tokens, logp = [], []
    for i in range(c["b"]):
        z = s["logits"][i].double()
        lp = torch.log_softmax(z / (temp[i] if temp[i] > 0 else 1.0), 0)
        if temp[i] <= 0:
            pick = int((z == z.max()).nonzero()[0, 0])
        else:
            p = lp.exp()
            order = torch.argsort(z, descending=True, stable=True)
            if 0 < top_k[i] < c["vocab"]:
                order = order[:int(top_k[i])]
            if top_p[i] < 1:
                upto = p[order].cumsum(0)
                order = order[:max(1, int((upto < top_p[i] * upto[-1]).sum()) + 1)]
            order = order[p[order] >= min_p[i] * p.max()]
            order = order.sort().values
            cdf = p[order].cumsum(0)
            pick = int(order[int((cdf <= u[i] * cdf[-1]).sum())])
        tokens.append(pick)
        logp.append(lp[pick])
    return {"tokens": _i32(tokens), "logp": torch.stack(logp)}


def _exact_lora(s):
    c = s["case"]
    r, ids = c["rank"], s["ids"].long()
    out = [t.double() for t in s["y0"]]
    for a in range(c["adapters"]):
        at = (ids == a).nonzero()[:, 0]
        for i in range(0, len(at), 512):
            rows = at[i:i + 512]
            for j, y in enumerate(out):
                low = s["x"][rows].double() @ s["a"][a, j * r:(j + 1) * r].double().T.contiguous()
                y[rows] += (low @ s["b"][j][a].double().T.contiguous()) * s["scale"][a].double()
    return {"y%d" % j: y for j, y in enumerate(out)}


def exact(case, seed):
    kinds = {"plan": _exact_plan, "rope": _exact_rope, "rope_kv": _exact_rope_kv, "sample": _exact_sample, "lora": _exact_lora}
    return kinds[case["kind"]](prepare(case, seed))
