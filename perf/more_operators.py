"""The operators on a cache in pages, as cases to measure.

Kinds:

  write   rows of a ragged batch of prompts go into their pages, normalised,
          rotated and quantised (smol_kv_pages_append), and come back as the
          values that the cache now stands for (smol_kv_pages_read), as a
          prompt's attention over its own cached rows needs them
  read    rows of cached prefixes come back (smol_kv_pages_read), as a chunk
          of a prompt behind them needs
  decode  one decode step's attention over pages of bf16 or of 8 bits
          (smol_attn_decode_paged)
  top     one decode step's attention over the pages that a bound on their
          scores selects (smol_attn_decode_paged_top)

A pool of pages of 64 rows holds, for each page and kv head,
  K       [hd / e][64][e], e = 16 codes or 8 bf16 numbers (16 bytes)
  V       codes [hd][64], or bf16 [2][hd][32]: rows of a page along a line, in
          the order of ORDER
  scales  fp32 [2][64], K's rows and V's (8 bits: a row is its codes times its
          scale)
  bounds  bf16 [2][hd], the lowest and the highest value of K's rows

`run` computes an operator with elementary torch operations in 32 bits (64 for
the scores that pages are chosen by) where `own` is false, and through the
library (smol_attn.py) where it is true. The 8-bit rows that a decode step
stores are returned as values: read back, which a server does not do after a
step. Keys are correlated within a page, queries have scores of a standard
deviation near 1.5.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6
PAGE = 64

# head layouts: (query heads, kv heads, head_dim, rope pairing, theta, per-head Q/K norm)
HEADS = {
    "qwen": (16, 8, 128, "neox", 1e6, True),           # Qwen3-ASR decoders
    "plain": (16, 8, 128, "neox", 1e6, False),         # the same without the per-head norm
    "mqa": (8, 1, 256, "interleaved", 1e4, False),     # Gemma-2B-style MQA
    "gemma": (8, 4, 256, "interleaved", 1e6, True),    # Gemma 3 style
    "small": (8, 4, 64, "neox", 1e6, True),
    "odd": (15, 5, 80, "neox", 1e4, False),            # 3 query heads a kv head, head_dim off the powers of two
}

# where a row of a page lies along V's line: rows 16 t + 4 g + i, t, g, i = 0 .. 3, by (g, t, i)
ORDER = {8: [r % 16 // 4 * 16 + r // 16 * 4 + r % 4 for r in range(64)],
         16: [r // 32 * 32 + r % 16 // 4 * 8 + r % 32 // 16 * 4 + r % 4 for r in range(64)]}


def listed():
    return [
        # a question's tokens behind a long document: latency
        dict(name="write_26_on_8192", op="write", heads="qwen", n_seq=1, pos=8192, len_lo=26, len_hi=26, bits=8,
             bf16=False),
        # prompts of several requests in one batch, projections in bf16, a bf16 pool
        dict(name="write_6_of_512", op="write", heads="gemma", n_seq=6, pos=0, len_lo=129, len_hi=512, bits=16, bf16=True),
        # a server's batch of long prompts: the largest
        dict(name="write_16_of_4096", op="write", heads="plain", n_seq=16, pos=0, len_lo=2000, len_hi=4096, bits=8,
             bf16=True),
        # a cached conversation in front of its next turn
        dict(name="read_1_of_1500", op="read", heads="small", n_seq=1, pos=0, len_lo=1500, len_hi=1500, bits=8, bf16=False),
        # cached documents in front of a batch of questions
        dict(name="read_8_of_8192", op="read", heads="qwen", n_seq=8, pos=64, len_lo=4000, len_hi=8192, bits=8, bf16=True),
        # one recording's transcript: latency
        dict(name="decode_1_of_1024", op="decode", heads="qwen", n_seq=1, len_lo=1024, len_hi=1024, bits=16, bf16=False,
             window=0, cap=0.0),
        # a served batch of conversations on a cache of 8 bits
        dict(name="decode_16_of_4160", op="decode", heads="qwen", n_seq=16, len_lo=3000, len_hi=4160, bits=8, bf16=False,
             window=0, cap=0.0),
        # one kv head for all, capped scores, bf16 projections
        dict(name="decode_mqa_24_of_8191", op="decode", heads="mqa", n_seq=24, len_lo=500, len_hi=8191, bits=16, bf16=True,
             window=0, cap=50.0),
        # a full batch of long conversations, 8 bits: the largest
        dict(name="decode_64_of_16384", op="decode", heads="plain", n_seq=64, len_lo=4000, len_hi=16384, bits=8, bf16=False,
             window=0, cap=0.0),
        # one long document, an eighth of its pages a step: latency
        dict(name="top_1_of_16384", op="top", heads="qwen", n_seq=1, len_lo=16384, len_hi=16384, bits=16, bf16=False, top=32,
             first=1, recent=2, cap=0.0),
        # a served batch of long documents, 8 bits
        dict(name="top_16_of_32768", op="top", heads="qwen", n_seq=16, len_lo=16000, len_hi=32768, bits=8, bf16=False, top=64,
             first=1, recent=4, cap=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.4)))))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode", "top"])
    hi = _log(rng, 1, {"write": 4096, "read": 8192, "decode": 16384, "top": 32768}[op])
    c = dict(op=op, heads=rng.choice(sorted(HEADS)), n_seq=_log(rng, 1, 64), len_lo=rng.randint(hi // 4 if op == "top" else 1, hi),
             len_hi=hi, bits=rng.choice([8, 8, 16]), bf16=rng.random() < 0.5)
    if op in ("write", "read"):
        c["pos"] = rng.choice([0, 0, rng.randint(1, 8192)])
    else:
        c["cap"] = rng.choice([0.0, 0.0, 50.0])
        if op == "decode":
            c["window"] = rng.choice([0, 0, _log(rng, 32, 8192)])
        else:
            c["top"] = _log(rng, 4, 128)
            c["first"], c["recent"] = rng.randint(0, 2), rng.randint(1, 2)
    # fewer sequences where a case would cost more than the largest listed one of its kind
    for unit in ("bytes", "flops"):
        most = max(work(k)[unit] for k in listed() if k["op"] == op)
        while work(c)[unit] > most and c["n_seq"] > 1:
            c["n_seq"] = (c["n_seq"] + 1) // 2
    return c


def work(c):
    """each stored row, bound and input read once, each output written once"""
    hq, hkv, hd = HEADS[c["heads"]][:3]
    n, mean = c["n_seq"], (c["len_lo"] + c["len_hi"]) / 2
    row = hkv * (2 * hd * c["bits"] // 8 + (8 if c["bits"] == 8 else 0))  # K and V of one stored row
    el = 2 if c["bf16"] else 4
    if c["op"] == "read":
        return {"bytes": n * mean * (row + 2 * hkv * hd * el), "flops": 0}
    if c["op"] == "write":
        return {"bytes": n * mean * (2 * hkv * hd * el + row + row + 2 * hkv * hd * el), "flops": 0}
    io = n * (hq * hd * (el + 4) + 2 * hkv * hd * el + row)
    seen = mean
    if c["op"] == "top":
        seen = min(mean, c["top"] * PAGE)
        if seen < mean:
            io += n * hkv * mean / PAGE * hd * 4
    elif c["window"]:
        seen = min(mean, c["window"] - 1)
    return {"bytes": n * seen * row + io, "flops": 4 * n * hq * hd * (seen + 1)}


# ------------------------------------------------------------------ inputs

_tables = {}


def _table(hd, theta, n):
    """The decoders' cos and sin rows [n][hd / 2] (fp32): 1 / theta^(2 d / hd) and its products with the positions
    are rounded to fp32, as the models' tables are; their cosines and sines are taken in 64 bits."""
    size = 1024
    while size < n:
        size *= 2
    if (hd, theta, size) not in _tables:
        e = np.arange(0, hd, 2, dtype=np.float32) / np.float32(hd)
        inv = np.float32(1) / (np.float64(theta) ** e.astype(np.float64)).astype(np.float32)
        ang = (np.arange(size, dtype=np.float32)[:, None] * inv[None, :]).astype(np.float64)
        _tables[hd, theta, size] = tuple(torch.from_numpy(f(ang).astype(np.float32)).to(DEV) for f in (np.cos, np.sin))
    return _tables[hd, theta, size]


def _outward(x, up):
    """fp32 numbers as the next bf16 below or above"""
    b = x.to(torch.bfloat16)
    bits = b.view(torch.int16)
    # one step away from zero where rounding went the wrong way on the side of x, one towards it on the other
    wrong = (b.float() < x) if up else (b.float() > x)
    step = torch.where((bits < 0) == up, -1, 1).to(torch.int16)
    return torch.where(wrong, bits + step, bits).view(torch.bfloat16)


def _inputs(c, seed):
    """the tensors of one case, alike for every side"""
    hq, hkv, hd, pairing, theta, norm = HEADS[c["heads"]]
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + 11)
    # lengths are the case's: outputs have the same shapes whatever the seed
    py = random.Random("%s %d %d %d" % (c["op"], c["n_seq"], c["len_lo"], c["len_hi"]))

    def normal(*shape, dtype=torch.float32, std=1.0):
        x = torch.empty(shape, dtype=dtype, device=DEV)
        x.normal_(0.0, std, generator=g)
        return x

    n, op, bits = c["n_seq"], c["op"], c["bits"]
    lens = [py.randint(c["len_lo"], c["len_hi"]) for _ in range(n)]
    lens[py.randrange(n)] = c["len_hi"]
    first = c["pos"] if op in ("write", "read") else 0
    ends = [first + l for l in lens] if op in ("write", "read") else [l + 1 for l in lens]
    need = [(e + PAGE - 1) // PAGE for e in ends]
    stride, total = max(need) + 2, sum(need)
    pages = total + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((n, stride), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    dt = torch.bfloat16 if c["bf16"] else torch.float32
    e = 16 if bits == 8 else 8
    ch = (hd + e - 1) // e
    live = (torch.arange(ch * e, device=DEV) < hd).view(ch, 1, e)  # the last piece of a head_dim that fills none is padded
    v_shape = (pages, hkv, hd, PAGE) if bits == 8 else (pages, hkv, 2, hd, PAGE // 2)
    k = normal(pages, hkv, ch, PAGE, e, std=0.7).add_(normal(pages, hkv, ch, 1, e, std=0.7)).mul_(live)
    if bits == 8:
        kp = k.mul_(42).round_().clamp_(-127, 127).to(torch.int8)
        vp = normal(*v_shape, std=42.0).round_().clamp_(-127, 127).to(torch.int8)
        scales = torch.exp(normal(pages, hkv, 2, PAGE, std=0.1)) / 42
        k = kp.float() * scales[:, :, 0, None, :, None]
    else:
        kp, vp, scales = k.to(torch.bfloat16), normal(*v_shape, dtype=torch.bfloat16), None
        k = kp.float()
    ext = torch.stack([_outward(k.amin(3), False), _outward(k.amax(3), True)], 2)
    bounds = ext.flatten(3)[..., :hd].contiguous()
    d = dict(kp=kp, vp=vp, scales=scales, bounds=bounds, table=table, pages=pages, lens=lens, inter=pairing == "interleaved",
             scale=hd ** -0.5 * (1.0 if norm else 1.5), q_norm=1.5 + normal(hd, std=0.1) if norm else None,
             k_norm=1.0 + normal(hd, std=0.1) if norm else None)
    if op in ("write", "read"):
        rows = sum(lens)
        starts = np.concatenate([[0], np.cumsum(lens)])
        seq = np.repeat(np.arange(n), lens)
        pos = np.arange(rows) - starts[seq] + first
        d["rows"], d["pos0"] = rows, torch.full((n,), first, dtype=torch.int32, device=DEV)
    else:
        rows, starts, seq, pos = n, np.arange(n + 1), np.arange(n), np.array(lens)
        d["pos0"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        d["q"] = normal(n, hq * hd, dtype=dt)
    d["starts"] = torch.from_numpy(starts.astype(np.int32)).to(DEV)
    d["seq"], d["pos"] = torch.from_numpy(seq).to(DEV), torch.from_numpy(pos).to(DEV)
    d["last"] = int(pos.max())
    if op != "read":
        d["k_new"], d["v_new"] = normal(rows, hkv * hd, dtype=dt), normal(rows, hkv * hd, dtype=dt)
        cos, sin = _table(hd, theta, d["last"] + 1)
        d["cos"], d["sin"] = cos[d["pos"]], sin[d["pos"]]
    return d


_kept = {}  # the context and the position tables that a program makes once


def _sa():
    import importlib
    sa = importlib.import_module("smol-genius_amd.smol_attn")
    if "ctx" not in _kept:
        _kept["ctx"] = sa.Context(0)
    return sa, _kept["ctx"]


def prepare(case, seed):
    c, d = case, _inputs(case, seed)
    d["case"] = c
    d["order"] = torch.tensor(ORDER[c["bits"]], device=DEV)
    if own:
        hq, hkv, hd, pairing, theta, _ = HEADS[c["heads"]]
        sa, ctx = _sa()
        d["pool"] = sa.KVPages(ctx, 1, d["pages"], hkv, hd, sa.INT8 if c["bits"] == 8 else sa.BF16)
        for name, view in zip(("kp", "vp", "scales", "bounds"), d["pool"].views(0)):
            if view is not None:
                view.copy_(d[name])
                d[name] = view
        key = (hd, theta, pairing)
        if key not in _kept:
            _kept[key] = sa.RopeTable(ctx, hd, theta, sa.ROPE_INTERLEAVED if d["inter"] else sa.ROPE_NEOX)
        _kept[key].ensure(d["table"].shape[1] * PAGE)
        d["rope"] = _kept[key]
    return d


# -------------------------------------------------------------- plain forms

def _normed(x, w):
    if w is None:
        return x
    return x * w / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)


def _rotated(x, cos, sin, inter):
    """x [n][heads][hd] by the table rows cos, sin [n][hd / 2]"""
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., 0::2], x[..., 1::2]) if inter else x.chunk(2, -1)
    y = (a * cos - b * sin, b * cos + a * sin)
    return torch.stack(y, -1).flatten(-2) if inter else torch.cat(y, -1)


def _codes(x):
    """8-bit codes of rows x [...][hd] and their scales"""
    top = x.abs().amax(-1, keepdim=True)
    codes = torch.round(x * (127.0 / top)).to(torch.int8)
    return codes, (top / 127.0).squeeze(-1)


def _pieces(x, e):
    """rows [n][kv][hd] as K's pieces [n][kv][hd / e][e], the last one padded"""
    pad = -x.shape[-1] % e
    return torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, e))


def _store(s, c, k, v):
    """rows k, v [n][kv][hd] (32 bits) into their pages, and the pages' bounds"""
    bits, hd = c["bits"], k.shape[-1]
    page, row = s["table"][s["seq"], s["pos"] // PAGE].long(), s["pos"] % PAGE
    at = s["order"][row]
    if bits == 8:
        (kq, ks), (vq, vs) = _codes(k), _codes(v)
        s["kp"][page, :, :, row] = _pieces(kq, 16)
        s["vp"][page, :, :, at] = vq
        s["scales"][page, :, 0, row], s["scales"][page, :, 1, row] = ks, vs
        kept = kq.float() * ks[..., None]
    else:
        kq, vq = k.to(torch.bfloat16), v.to(torch.bfloat16)
        s["kp"][page, :, :, row] = _pieces(kq, 8)
        s["vp"][page, :, at // 32, :, at % 32] = vq
        kept = kq.float()
    # bounds start anew with a page's first row
    lo, hi = s["bounds"][:, :, 0].float(), s["bounds"][:, :, 1].float()
    fresh = page[row == 0]
    lo[fresh], hi[fresh] = float("inf"), float("-inf")
    each = page[:, None, None].expand_as(kept)
    lo.scatter_reduce_(0, each, kept, "amin")
    hi.scatter_reduce_(0, each, kept, "amax")
    s["bounds"][:, :, 0], s["bounds"][:, :, 1] = _outward(lo, False), _outward(hi, True)


def _values(s, c, page, row):
    """stored rows [n][kv][hd] of K and V, 32 bits"""
    bits, hd = c["bits"], HEADS[c["heads"]][2]
    at = s["order"][row]
    k = s["kp"][page, :, :, row].float().flatten(-2)[..., :hd]
    if bits == 8:
        v = s["vp"][page, :, :, at].float()
        return k * s["scales"][page, :, 0, row][..., None], v * s["scales"][page, :, 1, row][..., None]
    return k, s["vp"][page, :, at // 32, :, at % 32].float()


def _back(s, c, dtype):
    page, row = s["table"][s["seq"], s["pos"] // PAGE].long(), s["pos"] % PAGE
    k, v = _values(s, c, page, row)
    return {"k": k.to(dtype).flatten(1), "v": v.to(dtype).flatten(1)}


def _state(s):
    """what the pool holds besides the rows: one tensor each, scales where there are any"""
    return {"bounds": s["bounds"]} if s["scales"] is None else {"bounds": s["bounds"], "scales": s["scales"]}


def _pages_of(s, c, pages, g=None):
    """K and V [...][kv][64][hd] of whole pages [...], 32 bits; with g: of kv head g alone, [...][64][hd]"""
    hd = HEADS[c["heads"]][2]
    pick = (lambda x: x[pages]) if g is None else (lambda x: x[pages, g])
    k = pick(s["kp"]).transpose(-3, -2).flatten(-2)[..., :hd].float()
    v = pick(s["vp"]) if c["bits"] == 8 else pick(s["vp"]).transpose(-3, -2).flatten(-2)
    v = v[..., s["order"]].float().transpose(-1, -2)
    if c["bits"] == 8:
        sc = pick(s["scales"])
        k, v = k * sc[..., 0, :, None], v * sc[..., 1, :, None]
    return k, v


def _attend(q, keys, vals, seen, k, v, scale, cap):
    """q [n][kv][G][hd] over keys, vals [n][kv][m][hd] where seen [n][kv or 1][m], and over the new row k, v [n][kv][hd]"""
    x = torch.cat([q @ keys.transpose(-1, -2), q @ k[..., None]], -1) * scale
    if cap > 0:
        x = torch.tanh(x / cap) * cap
    x[..., :-1].masked_fill_(~seen[:, :, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    return (x[..., :-1] @ vals + x[..., -1:] * v[:, :, None]) / x.sum(-1, keepdim=True)


def _step(s, c):
    hq, hkv, hd = HEADS[c["heads"]][:3]
    n = c["n_seq"]
    q = _rotated(_normed(s["q"].float().view(n, hq, hd), s["q_norm"]), s["cos"], s["sin"], s["inter"])
    k = _rotated(_normed(s["k_new"].float().view(n, hkv, hd), s["k_norm"]), s["cos"], s["sin"], s["inter"])
    return q.view(n, hkv, hq // hkv, hd), k, s["v_new"].float().view(n, hkv, hd)


def _stored(s, c):
    """what a decode step wrote: the pool's rows themselves where they are numbers, the new rows' values where they are codes"""
    if c["bits"] == 16:
        return {"k": s["kp"], "v": s["vp"]}
    return _back(s, c, torch.bfloat16)


def _run_decode(s, c):
    hkv = HEADS[c["heads"]][1]
    q, k, v = _step(s, c)
    n, held = c["n_seq"], (max(s["lens"]) + PAGE - 1) // PAGE
    keys, vals = _pages_of(s, c, s["table"][:, :held].clamp(min=0).long())  # [n][pages][kv][64][hd]
    keys, vals = (x.transpose(1, 2).flatten(2, 3) for x in (keys, vals))
    row, at = torch.arange(held * PAGE, device=DEV), s["pos"][:, None]
    seen = row < at
    if c["window"]:
        seen = seen & (row > at - c["window"])
    out = _attend(q, keys, vals, seen[:, None], k, v, s["scale"], c["cap"])
    _store(s, c, k, v)
    return {"out": out.reshape(n, -1), **_stored(s, c), **_state(s)}


def _run_top(s, c):
    hq, hkv, hd = HEADS[c["heads"]][:3]
    q, k, v = _step(s, c)
    n, top = c["n_seq"], c["top"]
    held = (max(s["lens"]) + PAGE - 1) // PAGE
    count = (s["pos"] + PAGE - 1)[:, None] // PAGE  # pages of each sequence
    page = s["table"][:, :held].clamp(min=0).long()
    # the bounds on the scores of a page's rows, summed over the heads, in 64 bits: which pages are chosen hangs on
    # differences as small as they come
    cos, sin = s["cos"].double(), s["sin"].double()
    q64 = _rotated(_normed(s["q"].double().view(n, hq, hd), None if s["q_norm"] is None else s["q_norm"].double()), cos, sin,
                   s["inter"]).view(n, hkv, -1, hd) * s["scale"]
    up, down = q64.clamp(min=0).sum(2), q64.clamp(max=0).sum(2)  # [n][kv][hd]
    b = s["bounds"][page].double()  # [n][pages][kv][2][hd]
    score = (b[..., 1, :] * up[:, None] + b[..., 0, :] * down[:, None]).sum(-1).transpose(1, 2)  # [n][kv][pages]
    j = torch.arange(held, device=DEV)
    score = score.masked_fill(((j < c["first"]) | (j >= count - c["recent"]))[:, None], float("inf"))
    score = score.masked_fill((j >= count)[:, None], float("-inf"))
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    best = torch.where(best < count[..., None], best, held)
    best = torch.nn.functional.pad(torch.sort(best, dim=-1).values, (0, top - best.shape[-1]), value=held)
    live = best < held
    at = torch.where(live, best, 0)
    of = page[:, None].expand(-1, hkv, -1).gather(2, at)  # [n][kv][top]
    keys, vals = _pages_of(s, c, of, torch.arange(hkv, device=DEV)[None, :, None])
    seen = live[..., None] & (at[..., None] * PAGE + torch.arange(PAGE, device=DEV) < s["pos"][:, None, None, None])
    out = _attend(q, keys.flatten(2, 3), vals.flatten(2, 3), seen.flatten(2), k, v, s["scale"], c["cap"])
    _store(s, c, k, v)
    return {"out": out.reshape(n, -1), "chosen": torch.where(live, best, -1).to(torch.int32), **_stored(s, c), **_state(s)}


def run(state):
    s, c = state, state["case"]
    dtype = torch.bfloat16
    if own:
        sa, ctx = _sa()
        pool, n = s["pool"], c["n_seq"]
        hq = HEADS[c["heads"]][0]
        if c["op"] == "write":
            sa.pages_append(pool, 0, s["rope"], s["table"], s["starts"], s["pos0"], s["k_new"], s["v_new"], k_norm=s["k_norm"],
                            eps=EPS)
        if c["op"] in ("write", "read"):
            k, v = sa.pages_read(pool, 0, s["table"], s["starts"], s["pos0"], s["rows"],
                                 dtype=dtype if c["bf16"] or c["op"] == "write" else torch.float32)
            return {"k": k, "v": v, **(_state(s) if c["op"] == "write" else {})}
        if c["op"] == "decode":
            out = {"out": sa.decode_paged(ctx, pool, 0, s["rope"], s["table"], s["pos0"], s["q"], s["k_new"], s["v_new"], hq,
                                          s["scale"], window=c["window"], cap=c["cap"], q_norm=s["q_norm"],
                                          k_norm=s["k_norm"], eps=EPS)}
        else:
            got, chosen = sa.decode_paged_top(ctx, pool, 0, s["rope"], s["table"], s["pos0"], s["q"], s["k_new"], s["v_new"],
                                              hq, s["scale"], c["top"], first=c["first"], recent=c["recent"], cap=c["cap"],
                                              q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
            out = {"out": got, "chosen": chosen}
        if c["bits"] == 16:
            return {**out, "k": s["kp"], "v": s["vp"], **_state(s)}
        k, v = sa.pages_read(pool, 0, s["table"], s["starts"], s["pos0"], n, dtype=dtype)
        return {**out, "k": k, "v": v, **_state(s)}
    if c["op"] == "read":
        return _back(s, c, dtype if c["bf16"] else torch.float32)
    if c["op"] == "write":
        hkv, hd = HEADS[c["heads"]][1:3]
        k = s["k_new"].float().view(-1, hkv, hd)
        k = _rotated(_normed(k, s["k_norm"]), s["cos"], s["sin"], s["inter"])
        _store(s, c, k, s["v_new"].float().view(-1, hkv, hd))
        return {**_back(s, c, dtype), **_state(s)}
    return (_run_decode if c["op"] == "decode" else _run_top)(s, c)


# ------------------------------------------------------------------ 64 bits

def _turn(x, w, cos, sin, inter):
    """heads [n][h][hd] in 64 bits: x w / sqrt(mean x^2 + eps), then the pairs as complex numbers times cos + i sin"""
    x = x.double()
    if w is not None:
        x = x * (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * w.double()
    by = torch.complex(cos.double(), sin.double())[:, None]
    if inter:
        return torch.view_as_real(torch.complex(x[..., 0::2].contiguous(), x[..., 1::2].contiguous()) * by).flatten(2)
    half = x.shape[2] // 2
    z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * by
    return torch.cat([z.real, z.imag], 2)


def _held(x, bits):
    """what a pool keeps of rows x [...][hd]: the values and their scales"""
    if bits == 16:
        return x.to(torch.bfloat16).double(), None
    unit = x.abs().amax(-1, keepdim=True) / 127
    return (x / unit).round() * unit, unit.squeeze(-1)


def _page64(d, c, page, kv):
    """rows [64][hd] of K and V of one page and kv head, in 64 bits"""
    hd = d["bounds"].shape[-1]
    k = torch.cat(list(d["kp"][page, kv].double()), -1)[:, :hd]
    v = d["vp"][page, kv].double()
    if c["bits"] == 8:
        v = torch.stack([v[:, i] for i in ORDER[8]])
        sc = d["scales"][page, kv].double()
        return k * sc[0][:, None], v * sc[1][:, None]
    return k, torch.stack([v[i // 32, :, i % 32] for i in ORDER[16]])


def _rows64(d, c, pages):
    """rows [kv][64 m][hd] of K and V of the pages listed, in 64 bits"""
    hd, m = d["bounds"].shape[-1], len(pages)
    k = d["kp"][pages].double().permute(1, 0, 3, 2, 4).reshape(d["kp"].shape[1], m * PAGE, -1)[..., :hd]
    v = d["vp"][pages].double()
    if c["bits"] == 16:
        v = v.permute(0, 1, 3, 2, 4).reshape(m, -1, hd, PAGE)
    back = torch.empty(PAGE, dtype=torch.long)
    for r, i in enumerate(ORDER[c["bits"]]):
        back[r] = i
    v = v[..., back.to(DEV)].permute(1, 0, 3, 2).reshape(-1, m * PAGE, hd)
    if c["bits"] == 8:
        sc = d["scales"][pages].double()
        k = k * sc[:, :, 0].permute(1, 0, 2).reshape(-1, m * PAGE, 1)
        v = v * sc[:, :, 1].permute(1, 0, 2).reshape(-1, m * PAGE, 1)
    return k, v


def _after64(c, d, k, v):
    """the pool after rows k, v [rows][kv][hd] (64 bits) went into it: the rows as stored, bounds and scales"""
    (kk, ks), (vv, vs) = _held(k, c["bits"]), _held(v, c["bits"])
    bounds = d["bounds"].double()
    scales = None if d["scales"] is None else d["scales"].double()
    table, pos = d["table"].cpu().numpy(), d["pos"].cpu().numpy()
    seq = d["seq"].cpu().numpy()
    page = table[seq, pos // PAGE]
    for i in range(c["n_seq"]):
        mine = np.flatnonzero(seq == i)
        for j in np.unique(pos[mine] // PAGE):
            r = mine[pos[mine] // PAGE == j]
            p, x = int(table[i, j]), kk[r[0]:r[-1] + 1]
            lo, hi = x.amin(0), x.amax(0)
            if pos[r[0]] % PAGE:
                lo, hi = torch.minimum(lo, bounds[p, :, 0]), torch.maximum(hi, bounds[p, :, 1])
            bounds[p, :, 0], bounds[p, :, 1] = lo, hi
    if scales is not None:
        pt, rt = torch.from_numpy(page.astype(np.int64)).to(DEV), d["pos"] % PAGE
        scales[pt, :, 0, rt], scales[pt, :, 1, rt] = ks, vs
    ans = {"bounds": bounds} if scales is None else {"bounds": bounds, "scales": scales}
    return kk, vv, page, ans


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    hq, hkv, hd = HEADS[c["heads"]][:3]
    table, lens = d["table"].cpu().numpy(), d["lens"]
    if c["op"] == "read":
        first, ks, vs = c["pos"], [], []
        for i, l in enumerate(lens):
            a, b = first // PAGE, (first + l + PAGE - 1) // PAGE
            k, v = _rows64(d, c, table[i, a:b].tolist())
            cut = slice(first - a * PAGE, first - a * PAGE + l)
            ks.append(k[:, cut].transpose(0, 1).reshape(l, -1))
            vs.append(v[:, cut].transpose(0, 1).reshape(l, -1))
        return {"k": torch.cat(ks), "v": torch.cat(vs)}
    k = _turn(d["k_new"].view(-1, hkv, hd), d["k_norm"], d["cos"], d["sin"], d["inter"])
    v = d["v_new"].double().view(-1, hkv, hd)
    kk, vv, page, ans = _after64(c, d, k, v)
    if c["op"] == "write":
        return {"k": kk.flatten(1), "v": vv.flatten(1), **ans}
    n, grp = c["n_seq"], hq // hkv
    q = _turn(d["q"].view(n, hq, hd), d["q_norm"], d["cos"], d["sin"], d["inter"]).view(n, hkv, grp, hd)
    out = torch.zeros((n, hkv, grp, hd), dtype=torch.float64, device=DEV)
    for i, l in enumerate(lens):
        m = (l + PAGE - 1) // PAGE
        keys, vals = _rows64(d, c, table[i, :m].tolist())
        seen = (torch.arange(m * PAGE, device=DEV) < l).expand(hkv, -1).clone()
        if c["op"] == "decode" and c["window"]:
            seen[:, :max(0, l - c["window"] + 1)] = False
        if c["op"] == "top" and m > c["top"]:
            b = d["bounds"][table[i, :m].tolist()].double()  # [m][kv][2][hd]
            for g in range(hkv):
                # sum over heads and dims of the larger of the products with either bound
                z = sum(torch.maximum(b[:, g, 0] * q[i, g, h], b[:, g, 1] * q[i, g, h]).sum(-1) for h in range(grp))
                z = z * d["scale"]
                fixed = [j for j in range(m) if j < c["first"] or j >= m - c["recent"]]
                rest = [j for j in range(m) if j not in set(fixed)]
                zs = z.tolist()
                rest.sort(key=lambda j: -zs[j])
                keep = torch.zeros(m, dtype=torch.bool)
                keep[fixed + rest[:c["top"] - len(fixed)]] = True
                seen[g] &= keep.to(DEV).repeat_interleave(PAGE)
        for g in range(hkv):
            kg = torch.cat([keys[g][seen[g]], k[i, g][None]])
            vg = torch.cat([vals[g][seen[g]], v[i, g][None]])
            z = q[i, g] @ kg.T.contiguous() * d["scale"]
            if c["cap"] > 0:
                z = c["cap"] * (z / c["cap"]).tanh()
            out[i, g] = z.softmax(-1) @ vg
    ans["out"] = out.reshape(n, -1)
    if c["op"] == "top":
        ans["chosen"] = None
    if c["bits"] == 8:
        return {**ans, "k": kk.flatten(1), "v": vv.flatten(1)}
    kp, vp = d["kp"].double(), d["vp"].double()
    for i, l in enumerate(lens):
        p, r = int(page[i]), l % PAGE
        piece = torch.zeros((hkv, kp.shape[2] * 8), dtype=torch.float64, device=DEV)
        piece[:, :hd] = kk[i]
        kp[p, :, :, r] = piece.view(hkv, -1, 8)
        a = ORDER[16][r]
        vp[p, :, a // 32, :, a % 32] = vv[i]
    return {**ans, "k": kp, "v": vp}
