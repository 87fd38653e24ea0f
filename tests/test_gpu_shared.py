"""Decode on a shared prefix, the scored decode step and cache eviction against plain 64-bit forms.

Bounds, derived before any run. A score is a sum of head_dim products of fp32
Q (three bf16 parts carry it whole) with exact bf16 K, so its error is that of
an fp32 sum, at most (hd + 8) 2^-24 sum |q k| scale with the rotation, the norm
and the scaling (about eight roundings). With scores of at most s_max in
magnitude and a probability p carried as two bf16 parts (bf16 has 8 significant
bits, so half a step is at most 2^-8 of a value: the first part leaves 2^-8 of
p, the second 2^-8 of that: 2^-16) and a sum of n terms, p's relative error is
at most
    e = 2 (hd + 16) 2^-24 a_max + 2^-16 + 2^-21,
a_max = max_j scale sum_d |q_d k_jd| (the exp and the sums of at most 64 chunks
of a few partial sums each add less than 2^-21), so
    |out - exact| <= 2 e sum_j p_j |v_j| + 2^-22 |exact|
(numerator and denominator each off by e), and a mass is off by 2 e times itself
for each addition. Appended rows are the exact ones rounded to bf16 (half a
step, 2^-8 of the value), plus what the fp32 norm and rotation may be off by:
2^-20 of the row's norm.
"""
import math

import numpy as np
import pytest

from conftest import pkg  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

EPS = 1e-6


@pytest.fixture(scope="module")
def sa():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from smol_genius_amd import smol_attn
    smol_attn.load()
    return smol_attn


@pytest.fixture(scope="module")
def ctx(sa):
    c = sa.Context(0)
    yield c
    c.close()


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(g, *shape, bf16=False, std=1.0):
    x = torch.randn(shape, generator=g) * std
    return x.to(torch.bfloat16) if bf16 else x


class Cache:
    """a device cache and its rows on the host, every row of every slot filled (rows past a length are never zeros)"""

    def __init__(self, sa, ctx, n_slots, hkv, hd, rows, g, layers=2, layer=1):
        self.kv = sa.KVCache(ctx, layers, n_slots, hkv, hd, rows)
        self.layer = layer
        self.k = normal(g, n_slots, hkv, self.kv.capacity, hd, bf16=True)
        self.v = normal(g, n_slots, hkv, self.kv.capacity, hd, bf16=True)
        self.push()

    def push(self):
        kt, vt = self.kv.views(self.layer)
        kt.copy_(self.k)
        ns, hkv, cap, hd = self.k.shape
        vt.copy_(self.v.view(ns, hkv, cap // 32, 32, hd).transpose(-1, -2))

    def pull(self):
        kt, vt = self.kv.views(self.layer)
        return kt.cpu(), vt.transpose(-1, -2).reshape(self.k.shape).cpu()


def table(sa, hd, theta, inter, pos):
    """cos and sin rows of the library's own table, in 64 bits"""
    c, s = zip(*(sa.rope_fill_host(p, 1, hd, theta, 1 if inter else 0) for p in pos))
    return torch.from_numpy(np.concatenate(c)).double(), torch.from_numpy(np.concatenate(s)).double()


def turned(x, w, rope, inter):
    """heads x [n, h, hd]: RMSNorm by w (None: none), rotation by the rows of rope (None: none), in 64 bits"""
    x = x.double()
    if w is not None:
        x = x * w.double() / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    if rope is None:
        return x
    c, s = rope[0][:, None], rope[1][:, None]
    if inter:
        y = torch.stack([-x[..., 1::2], x[..., 0::2]], -1).flatten(-2)
    else:
        a, b = x.chunk(2, -1)
        y = torch.cat([-b, a], -1)
    return x * c + y * s


def attend(q, k, v, scale, cap):
    """q [G, hd], k, v [m, hd] in 64 bits: out, weights, and sum_j p_j |v_j| with the largest scale sum |q k|"""
    z = q @ k.T * scale
    if cap:
        z = cap * torch.tanh(z / cap)
    p = torch.softmax(z, -1)
    a = (q.abs() @ k.abs().T * scale).max()
    return p @ v, p, p @ v.abs(), float(a)


def err(hd, a_max):
    return 2 * (hd + 16) * 2.0 ** -24 * a_max + 2.0 ** -16 + 2.0 ** -21


def check_rows(got_k, got_v, cache, slots, lens, k64, v64):
    """the appended rows are the exact ones in bf16, and nothing else of the layer changed"""
    hk, hv = cache.k.clone(), cache.v.clone()
    for i, (s, l) in enumerate(zip(slots, lens)):
        n = k64[i].norm(dim=-1, keepdim=True)
        assert ((got_k[s, :, l].double() - k64[i]).abs() <= 2.0 ** -8 * k64[i].abs() + 2.0 ** -20 * n).all()
        assert torch.equal(got_v[s, :, l], v64[i].float().to(torch.bfloat16))
        hk[s, :, l], hv[s, :, l] = got_k[s, :, l], got_v[s, :, l]
    assert torch.equal(hk.view(torch.int16), got_k.view(torch.int16))
    assert torch.equal(hv.view(torch.int16), got_v.view(torch.int16))


class Shared:
    """one shared decode step's inputs, its call and its check"""

    def __init__(self, sa, ctx, hq, hkv, hd, lens, prefix, inter=False, norm=True, bf16=False, window=0, cap=0.0, rope=True,
                 seed=1, std=1.0, same_cache=False):
        g = gen(seed)
        self.__dict__.update(sa=sa, ctx=ctx, hq=hq, hkv=hkv, hd=hd, lens=list(lens), prefix=prefix, inter=inter, window=window,
                             cap=cap)
        n = self.n = len(self.lens)
        self.scale = hd ** -0.5
        self.slots = [int(s) for s in torch.randperm(n + 2, generator=g)[:n]]
        if same_cache:
            self.own = Cache(sa, ctx, n + 3, hkv, hd, max(max(lens) + 1, prefix), g)
            self.pre, self.p_slot = self.own, n + 2
        else:
            self.own = Cache(sa, ctx, n + 2, hkv, hd, max(lens) + 1, g)
            self.pre, self.p_slot = Cache(sa, ctx, 2, hkv, hd, max(prefix, 1), g), 1
        self.q = normal(g, n, hq * hd, bf16=bf16, std=std)
        self.k = normal(g, n, hkv * hd, bf16=bf16)
        self.v = normal(g, n, hkv * hd, bf16=bf16)
        self.qw = 1.5 + 0.1 * normal(g, hd) if norm else None
        self.kw = 1.0 + 0.1 * normal(g, hd) if norm else None
        self.theta = 1e4
        self.rope = sa.RopeTable(ctx, hd, self.theta, 1 if inter else 0) if rope else None

    def call(self, **kw):
        d = lambda t: None if t is None else t.cuda()  # noqa: E731
        if not hasattr(self, "dev"):
            self.dev = [d(t) for t in (self.q, self.k, self.v)], [d(self.qw), d(self.kw)]
        (q, k, v), (qw, kw_) = self.dev
        return self.sa.decode_shared(self.ctx, self.pre.kv, self.p_slot, self.prefix, self.own.kv, self.own.layer, self.rope,
                                     self.slots, self.lens, q, k, v, self.hq, self.scale, window=self.window, cap=self.cap,
                                     q_norm=qw, k_norm=kw_, eps=EPS, **kw)

    def rows64(self):
        n, hd = self.n, self.hd
        rope = table(self.sa, hd, self.theta, self.inter, [self.prefix + l for l in self.lens]) if self.rope else None
        return (turned(self.q.view(n, self.hq, hd), self.qw, rope, self.inter),
                turned(self.k.view(n, self.hkv, hd), self.kw, rope, self.inter), self.v.double().view(n, self.hkv, hd))

    def check(self, out, rows=True):
        q, k, v = self.rows64()
        G = self.hq // self.hkv
        out = out.cpu().double().view(self.n, self.hkv, G, self.hd)
        worst = 0.0
        for i, (s, l) in enumerate(zip(self.slots, self.lens)):
            first = max(0, self.prefix + l - self.window + 1) if self.window else 0
            for h in range(self.hkv):
                P = self.prefix
                kk = torch.cat([self.pre.k[self.p_slot, h, :P].double(), self.own.k[s, h, :l].double(), k[i, h:h + 1]])[first:]
                vv = torch.cat([self.pre.v[self.p_slot, h, :P].double(), self.own.v[s, h, :l].double(), v[i, h:h + 1]])[first:]
                o, _, pv, a = attend(q[i].view(self.hkv, G, self.hd)[h], kk, vv, self.scale, self.cap)
                assert torch.isfinite(out[i, h]).all(), (i, h)
                tol = 2 * err(self.hd, a) * pv + 2.0 ** -22 * o.abs()
                worst = max(worst, float(((out[i, h] - o).abs() / tol).max()))
        print("shared hq %d hkv %d hd %d prefix %d lens %s: %.3f of the bound" % (self.hq, self.hkv, self.hd, self.prefix,
                                                                                  self.lens[:6], worst), flush=True)
        assert worst <= 1.0
        if rows:
            gk, gv = self.own.pull()
            check_rows(gk, gv, self.own, self.slots, self.lens, k, v)


SHARED = [
    # one row, an empty cache, an empty prefix
    dict(hq=4, hkv=2, hd=64, lens=[0], prefix=0),
    dict(hq=4, hkv=2, hd=64, lens=[0], prefix=1),
    dict(hq=4, hkv=2, hd=64, lens=[5], prefix=0),
    dict(hq=2, hkv=2, hd=72, lens=[0, 1, 31, 32, 33], prefix=31, inter=True),
    dict(hq=15, hkv=5, hd=80, lens=[63, 64, 65], prefix=128, norm=False),
    dict(hq=6, hkv=1, hd=96, lens=[100, 0, 7], prefix=129, bf16=True),
    dict(hq=16, hkv=8, hd=128, lens=[17, 300, 1, 0, 128, 127], prefix=500),
    dict(hq=16, hkv=8, hd=128, lens=[3, 9], prefix=2049, rope=False),
    # more rows a kv head than one tile, an odd number of them
    dict(hq=8, hkv=1, hd=256, lens=[200, 0, 31, 77, 5], prefix=1000, inter=True, bf16=True, cap=30.0),
    dict(hq=12, hkv=4, hd=128, lens=list(range(0, 46, 2)), prefix=700, cap=50.0),
    # more than 32 rows a kv head: 64 rows share the prefix's slabs, a last block of one row, less than a slab
    dict(hq=8, hkv=2, hd=128, lens=list(range(0, 34, 2)) + [100], prefix=1000),
    dict(hq=8, hkv=2, hd=64, lens=[i % 7 for i in range(33)], prefix=77, norm=False, inter=True),
    dict(hq=13, hkv=1, hd=64, lens=[1, 0, 5, 9, 40], prefix=5, cap=20.0),
    dict(hq=8, hkv=1, hd=256, lens=[0, 3, 64, 10, 7, 9, 200, 1, 5], prefix=523, inter=True, cap=30.0),
    dict(hq=8, hkv=1, hd=128, lens=[0, 10, 40, 200, 33, 7, 8, 9, 100], prefix=300, window=150),
    dict(hq=15, hkv=5, hd=96, lens=[2] * 12, prefix=200, bf16=True),
    # fifteen heads a kv head, and sixteen: the new key takes the sixteenth column
    dict(hq=15, hkv=1, hd=64, lens=[40, 0, 3], prefix=90),
    dict(hq=16, hkv=1, hd=72, lens=[40, 0], prefix=31, inter=True),
    # more heads a kv head than one tile
    dict(hq=34, hkv=2, hd=64, lens=[40, 0, 3], prefix=90),
    dict(hq=20, hkv=1, hd=256, lens=[10, 50], prefix=33, norm=False, inter=True),
    # windows: inside the own rows, across the prefix's end, different first keys a row
    dict(hq=4, hkv=2, hd=128, lens=[0, 10, 40, 200, 33], prefix=300, window=1),
    dict(hq=4, hkv=2, hd=128, lens=[0, 10, 40, 200, 33], prefix=300, window=50),
    dict(hq=4, hkv=2, hd=64, lens=[0, 10, 40, 200, 33, 7, 8, 9, 100], prefix=300, window=256),
    dict(hq=4, hkv=2, hd=80, lens=[0, 600, 40], prefix=300, window=5000),
    # sharp scores
    dict(hq=4, hkv=2, hd=128, lens=[60, 0, 200], prefix=400, std=8.0, norm=False),
    # sequences past what the kernel arguments hold
    dict(hq=2, hkv=1, hd=64, lens=[i % 5 for i in range(131)], prefix=70),
    dict(hq=4, hkv=2, hd=64, lens=[70, 3], prefix=65, same_cache=True),
]


@pytest.mark.parametrize("c", SHARED, ids=lambda c: "%d-%d-%d-p%d-n%d-w%d" % (c["hq"], c["hkv"], c["hd"], c["prefix"],
                                                                              len(c["lens"]), c.get("window", 0)))
def test_shared(sa, ctx, c):
    s = Shared(sa, ctx, **c)
    s.check(s.call())


def test_shared_long_prefix(sa, ctx):
    """more prefix than a chunk a workgroup, and a call on the same state again"""
    s = Shared(sa, ctx, 8, 2, 64, [600, 0, 30], 20000)
    a = s.call().clone()
    s.check(a)
    assert torch.equal(a, s.call())


@pytest.mark.parametrize("c", [
    dict(hq=4, hkv=2, hd=64, lens=[3] * 30 + [4000] + [i % 50 for i in range(30)], prefix=100),
    dict(hq=8, hkv=2, hd=128, lens=[20] * 140 + [3000], prefix=64, window=700),
    dict(hq=20, hkv=1, hd=80, lens=[2900] + [40] * 64, prefix=0),
], ids=["61", "141-window", "65-no-prefix"])
def test_shared_one_long_among_short(sa, ctx, c):
    """one sequence's own rows are many chunks, the others' one each"""
    s = Shared(sa, ctx, **c)
    a = s.call().clone()
    s.check(a)
    assert torch.equal(a, s.call())


@pytest.mark.parametrize("slabs", [-5, 1, 4, 7, 64, 2 ** 30, 2 ** 31 - 1])
def test_forced_slabs(sa, slabs):
    c2 = sa.Context(0)
    c2.set_option(sa.OPT_DEC_SLABS, slabs)
    s = Shared(sa, c2, 8, 2, 128, [3, 700, 0, 64] * 3, 1100, window=900)
    s.check(s.call())
    z = Scored(sa, c2, 4, 2, 64, [900, 0, 33])
    m, p = z.arrays()
    z.check(z.call(m, p), m, p)
    del s, z
    c2.close()


def test_shared_equals_decode(sa, ctx):
    """the batch's step on a shared prefix is the decode step of sequences that hold the prefix themselves"""
    s = Shared(sa, ctx, 8, 4, 128, [40, 0, 5], 333)
    out = s.call()
    kv = sa.KVCache(ctx, 1, 3, 4, 128, 512)
    kt, vt = kv.views(0)
    for i, (sl, l) in enumerate(zip(s.slots, s.lens)):
        rk = torch.cat([s.pre.k[s.p_slot, :, :333], s.own.k[sl, :, :l]], 1)
        rv = torch.cat([s.pre.v[s.p_slot, :, :333], s.own.v[sl, :, :l]], 1)
        flat = lambda t: t.transpose(0, 1).reshape(333 + l, -1).contiguous().cuda()  # noqa: E731
        kv.write(0, i, 0, flat(rk), flat(rv))
    (q, k, v), (qw, kw) = s.dev
    want = sa.decode(ctx, kv, 0, s.rope, [0, 1, 2], [333 + l for l in s.lens], q, k, v, 8, s.scale, q_norm=qw, k_norm=kw,
                     eps=EPS)
    # both within their own bounds of the exact result; the decode step carries Q in 17 bits
    assert (out - want).abs().max() <= 2e-3


def test_shared_stale_and_foreign_rows(sa, ctx):
    """NaN and infinity in rows past a length, past the prefix, in other slots and layers reach nothing; in a visible
    row they reach the sequence that sees it and no other"""
    s = Shared(sa, ctx, 4, 2, 128, [37, 5, 64], 77)
    clean = s.call().clone()
    bad = [float("nan"), float("inf"), -float("inf")]
    for i in range(s.own.k.shape[0]):
        for r in range(s.own.k.shape[2]):
            if i not in s.slots or r >= s.lens[s.slots.index(i)]:
                s.own.k[i, :, r], s.own.v[i, :, r] = bad[r % 3], bad[(r + 1) % 3]
    s.pre.k[s.p_slot, :, 77:], s.pre.v[s.p_slot, :, 77:] = float("nan"), float("inf")
    s.pre.k[0], s.pre.v[0] = float("nan"), float("nan")
    s.own.push()
    s.pre.push()
    assert torch.equal(clean, s.call())
    s.own.v[s.slots[1], :, 2] = float("inf")
    s.own.push()
    out = s.call()
    assert torch.equal(out[[0, 2]], clean[[0, 2]]) and not torch.isfinite(out[1]).any()


@pytest.mark.parametrize("heads", [(4, 2, 64), (28, 2, 64), (12, 3, 96)])
def test_shared_window_keeps_rows_apart(sa, ctx, heads):
    """a value that is not finite, in a prefix row that one sequence's window has left and another's has not"""
    s = Shared(sa, ctx, *heads, [0, 30, 60], 200, window=100)
    clean = s.call().clone()
    # rows seen: from 101, 131 and 161 on
    s.pre.v[s.p_slot, :, 140] = float("nan")
    s.pre.k[s.p_slot, :, 120] = float("inf")
    s.pre.push()
    out = s.call()
    assert torch.equal(out[2], clean[2])
    assert not torch.isfinite(out[0]).any() and not torch.isfinite(out[1]).any()


@pytest.mark.parametrize("hd,inter", [(64, False), (72, True), (128, False), (256, True)])
def test_shared_weights_off_sixteen_bytes(sa, ctx, hd, inter):
    """norm weights that begin four bytes into a buffer (their alignment is a float's)"""
    s = Shared(sa, ctx, 4, 2, hd, [30, 0, 65], 77, inter=inter)
    out = s.call().clone()
    for i, w in enumerate((s.qw, s.kw)):
        buf = torch.zeros(hd + 1, device="cuda")
        buf[1:] = w.cuda()
        s.dev[1][i] = buf[1:]
        assert buf[1:].data_ptr() % 16 == 4
    assert torch.equal(out, s.call())


def test_shared_grows_the_cache(sa, ctx):
    s = Shared(sa, ctx, 4, 2, 64, [63, 10], 50)
    assert s.own.kv.capacity == 64
    s.lens = [64, 10]
    out = s.call()
    assert s.own.kv.capacity == 128
    s.check(out, rows=False)


def test_shared_other_stream(sa):
    """a context on a stream of its own, behind work that fills the inputs there"""
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        c2 = sa.Context(0)
        s = Shared(sa, c2, 4, 2, 128, [30, 3], 300)
        out = s.call()
    st.synchronize()
    s.check(out)
    del s
    c2.close()


def test_shared_refusals(sa, ctx):
    s = Shared(sa, ctx, 4, 2, 64, [3, 4], 20)
    s.call()
    (q, k, v), (qw, kw) = s.dev
    L = sa.load()
    import ctypes

    def rc(prefix=None, p_slot=1, p_len=20, kv=None, layer=1, slots=None, lens=(3, 4), n=2, hq=4, dtype=0, qp=None, eps=EPS):
        sl = np.array(s.slots if slots is None else slots, np.int32)
        le = np.array(lens, np.int32)
        ip = ctypes.POINTER(ctypes.c_int)
        out = torch.empty(2, 256, device="cuda")
        return L.smol_attn_decode_shared(ctx.h, (prefix or s.pre.kv).h, p_slot, p_len, (kv or s.own.kv).h, layer, s.rope.h, n,
                                         sl.ctypes.data_as(ip), le.ctypes.data_as(ip), qp or q.data_ptr(), k.data_ptr(),
                                         v.data_ptr(), dtype, hq, s.scale, 0, 0.0, None, qw.data_ptr(), eps, out.data_ptr())
    assert rc() == 0
    assert rc(p_slot=2) == -1 and rc(p_slot=-1) == -1
    assert rc(p_len=-1) == -1 and rc(p_len=65) == -1
    assert rc(layer=2) == -1 and rc(layer=-1) == -1
    assert rc(slots=[0, 0]) == -1 and rc(slots=[0, 9]) == -1
    assert rc(lens=(3, -1)) == -1 and rc(lens=(3, 2 ** 31 - 70)) == -1
    assert rc(n=0) == -1 and rc(hq=5) == -1 and rc(dtype=2) == -1
    assert rc(qp=q.data_ptr() + 4) == -1
    assert rc(eps=-1.0) == -1 and rc(eps=float("nan")) == -1
    assert rc(prefix=s.own.kv, p_slot=s.slots[0], p_len=4) == -1
    other = sa.KVCache(ctx, 2, 2, 1, 64, 64)
    assert rc(prefix=other) == -1
    c2 = sa.Context(0)
    foreign = sa.KVCache(c2, 2, 4, 2, 64, 64)
    assert rc(prefix=foreign) == -1 and rc(kv=foreign) == -1
    with pytest.raises(sa.SmolAttnError):
        sa.decode_shared(ctx, s.pre.kv, 1, 20, s.own.kv, 1, s.rope, s.slots, [3], q, k, v, 4, s.scale)
    with pytest.raises(sa.SmolAttnError):
        sa.decode_shared(ctx, s.pre.kv, 1, 20, s.own.kv, 1, s.rope, s.slots, s.lens, q[:, :128], k, v, 4, s.scale)
    with pytest.raises(sa.SmolAttnError):
        sa.decode_shared(ctx, s.pre.kv, 1, 20, s.own.kv, 1, s.rope, s.slots, s.lens, q, k.to(torch.bfloat16), v, 4, s.scale)
    ctx.synchronize()
    s.check(s.call(), rows=False)
    foreign.close()
    c2.close()


# ------------------------------------------------------------------- scored

class Scored:
    def __init__(self, sa, ctx, hq, hkv, hd, rows, inter=False, norm=True, bf16=False, cap=0.0, decay=1.0, seed=2, gap=3):
        g = gen(seed)
        self.__dict__.update(sa=sa, ctx=ctx, hq=hq, hkv=hkv, hd=hd, rows=list(rows), inter=inter, cap=cap, decay=decay)
        n = self.n = len(self.rows)
        self.scale = hd ** -0.5
        self.slots = [int(s) for s in torch.randperm(n + 2, generator=g)[:n]]
        self.own = Cache(sa, ctx, n + 2, hkv, hd, max(rows) + 1, g)
        self.pos = [gap * r + 1 for r in rows]
        self.q, self.k, self.v = (normal(g, n, h * hd, bf16=bf16) for h in (hq, hkv, hkv))
        self.qw = 1.5 + 0.1 * normal(g, hd) if norm else None
        self.kw = 1.0 + 0.1 * normal(g, hd) if norm else None
        self.theta = 1e6
        self.rope = sa.RopeTable(ctx, hd, self.theta, 1 if inter else 0)
        stride = max(rows) + 1 + seed % 3
        self.mass = normal(g, n + 2, hkv, stride).abs()
        for s, r in zip(self.slots, rows):
            self.mass[s, :, r:] = float("nan")  # rows that hold nothing yet
        if decay == 0.0:
            self.mass[:] = float("nan")
        self.row_pos = torch.randint(0, 9999, (n + 2, hkv, stride), generator=g, dtype=torch.int32)

    def arrays(self):
        return self.mass.cuda(), self.row_pos.cuda()

    def call(self, mass, row_pos, **kw):
        d = lambda t: None if t is None else t.cuda()  # noqa: E731
        if not hasattr(self, "dev"):
            self.dev = [d(t) for t in (self.q, self.k, self.v)], [d(self.qw), d(self.kw)]
        (q, k, v), (qw, kw_) = self.dev
        return self.sa.decode_scored(self.ctx, self.own.kv, 1, self.rope, self.slots, self.rows, self.pos, q, k, v, self.hq,
                                     self.scale, mass, row_pos, decay=self.decay, cap=self.cap, q_norm=qw, k_norm=kw_,
                                     eps=EPS, **kw)

    def check(self, out, mass, row_pos):
        n, hd, G = self.n, self.hd, self.hq // self.hkv
        rope = table(self.sa, hd, self.theta, self.inter, self.pos)
        q = turned(self.q.view(n, self.hq, hd), self.qw, rope, self.inter)
        k = turned(self.k.view(n, self.hkv, hd), self.kw, rope, self.inter)
        v = self.v.double().view(n, self.hkv, hd)
        out, mass, row_pos = out.cpu().double().view(n, self.hkv, G, hd), mass.cpu(), row_pos.cpu()
        want_pos = self.row_pos.clone()
        untouched = torch.ones_like(mass, dtype=torch.bool)
        for i, (s, r) in enumerate(zip(self.slots, self.rows)):
            want_pos[s, :, r] = self.pos[i]
            untouched[s, :, :r + 1] = False
            for h in range(self.hkv):
                kk = torch.cat([self.own.k[s, h, :r].double(), k[i, h:h + 1]])
                vv = torch.cat([self.own.v[s, h, :r].double(), v[i, h:h + 1]])
                o, p, pv, a = attend(q[i].view(self.hkv, G, hd)[h], kk, vv, self.scale, self.cap)
                e = err(hd, a)
                assert ((out[i, h] - o).abs() <= 2 * e * pv + 2.0 ** -22 * o.abs()).all()
                w = p.sum(0)
                had = self.mass[s, h, :r + 1].double() * self.decay
                had[r] = 0.0
                if self.decay == 0.0:
                    had[:] = 0.0
                got = mass[s, h, :r + 1].double()
                # decay, the sum over the heads and the addition round once each
                assert ((got - had - w).abs() <= 2 * e * w + (G + 3) * 2.0 ** -24 * (had + w)).all()
        assert torch.equal(row_pos, want_pos)
        a, b = mass.view(torch.int32)[untouched], self.mass.view(torch.int32)[untouched]
        assert torch.equal(a, b)
        gk, gv = self.own.pull()
        check_rows(gk, gv, self.own, self.slots, self.rows, k, v)


@pytest.mark.parametrize("c", [
    dict(hq=4, hkv=2, hd=64, rows=[0]),
    dict(hq=4, hkv=2, hd=64, rows=[1, 0, 31, 32, 33], decay=0.0),
    dict(hq=15, hkv=5, hd=80, rows=[100, 1023, 1024, 1025], norm=False, bf16=True),
    dict(hq=16, hkv=8, hd=128, rows=[1024, 3, 2100], decay=0.9),
    dict(hq=8, hkv=1, hd=256, rows=[300, 7], inter=True, cap=30.0),
    dict(hq=3, hkv=3, hd=72, rows=[129, 64]),
    dict(hq=20, hkv=1, hd=96, rows=[40, 500], decay=0.0, cap=50.0),
    dict(hq=2, hkv=1, hd=64, rows=[i % 40 for i in range(130)]),
    # more heads a kv head than the weights' workgroups hold at once
    dict(hq=520, hkv=1, hd=64, rows=[40, 0]),
], ids=lambda c: "%d-%d-%d-%s" % (c["hq"], c["hkv"], c["hd"], "_".join(map(str, c["rows"][:4]))))
def test_scored(sa, ctx, c):
    s = Scored(sa, ctx, **c)
    m, p = s.arrays()
    s.check(s.call(m, p), m, p)


def test_scored_long(sa, ctx):
    s = Scored(sa, ctx, 4, 1, 64, [40000, 17], gap=1)
    m, p = s.arrays()
    s.check(s.call(m, p), m, p)


def test_scored_one_long_among_short(sa, ctx):
    s = Scored(sa, ctx, 2, 2, 64, [5] * 70 + [6000], gap=1)
    m, p = s.arrays()
    s.check(s.call(m, p), m, p)


@pytest.mark.parametrize("long", [1100, 4100])
def test_scored_many_pairs(sa, ctx, long):
    """more (sequence, kv head) pairs than there are workgroups to add weights up: each takes several runs of rows. The data
    is made on the device; the longest sequences and some others are checked"""
    n, hkv, hq, hd = 4200 * 1100 // long // 8, 8, 16, 64
    rows = [long if i in (0, n - 1) else i % 70 for i in range(n)]
    kv = sa.KVCache(ctx, 1, n, hkv, hd, long + 1)
    torch.manual_seed(5)
    kt, vt = kv.views(0)
    kt.normal_()
    vt.normal_()
    q, k, v = (torch.randn(n, h * hd, device="cuda") for h in (hq, hkv, hkv))
    mass = torch.rand(n, hkv, long + 3, device="cuda")
    row_pos = torch.zeros(n, hkv, long + 3, dtype=torch.int32, device="cuda")
    had = mass.clone()
    out = sa.decode_scored(ctx, kv, 0, None, list(range(n)), rows, rows, q, k, v, hq, hd ** -0.5, mass, row_pos, decay=0.5)
    assert torch.isfinite(out).all()
    for i in (0, 1, 69, n // 2, n - 1):
        r = rows[i]
        assert torch.equal(mass[i, :, r + 1:], had[i, :, r + 1:]) and (row_pos[i, :, r] == r).all()
        for h in range(hkv):
            kk = torch.cat([kt[i, h, :r].double(), k[i].view(hkv, hd)[h:h + 1].double()])
            vv = torch.cat([vt[i, h].transpose(1, 2).reshape(-1, hd)[:r].double(), v[i].view(hkv, hd)[h:h + 1].double()])
            o, p, pv, a = attend(q[i].view(hkv, 2, hd)[h].double(), kk, vv, hd ** -0.5, 0.0)
            e = err(hd, a)
            assert ((out[i].view(hkv, 2, hd)[h] - o).abs() <= 2 * e * pv + 2.0 ** -22 * o.abs()).all()
            w = p.sum(0)
            old = 0.5 * had[i, h, :r + 1].double()
            old[r] = 0.0
            assert ((mass[i, h, :r + 1] - old - w).abs() <= 2 * e * w + 5 * 2.0 ** -24 * (old + w)).all()
    kv.close()


def test_scored_refusals(sa, ctx):
    s = Scored(sa, ctx, 4, 2, 64, [10, 5])
    m, p = s.arrays()
    good = s.call(m, p).clone()
    for bad in (dict(m=m[:, :, :10].contiguous(), p=p[:, :, :10].contiguous()), dict(m=m.double(), p=p), dict(m=m, p=p.long()),
                dict(m=m[:1].contiguous(), p=p[:1].contiguous()), dict(m=m.transpose(1, 2), p=p)):
        with pytest.raises(sa.SmolAttnError):
            s.call(bad["m"], bad["p"])
    for field, value in (("decay", -1.0), ("decay", float("nan")), ("decay", float("inf")), ("pos", [-1, 3]),
                         ("rows", [-1, 3]), ("slots", [1, 1]), ("slots", [0, 4])):
        keep = getattr(s, field)
        setattr(s, field, value)
        with pytest.raises(sa.SmolAttnError):
            s.call(m, p)
        setattr(s, field, keep)
    with pytest.raises(sa.SmolAttnError, match="overlap"):
        s.call(m, m.view(torch.int32))
    # tables do not grow to any position, nor caches to any length: neither loops nor allocates
    keep = s.pos
    for far in (2 ** 22, 2 ** 30 + 1, 2 ** 31 - 70):
        s.pos = [far, 3]
        with pytest.raises(sa.SmolAttnError, match="table"):
            s.call(m, p)
    s.pos = keep
    (q, k, v), (qw, kw_) = s.dev
    for far in (2 ** 24, 2 ** 30 + 1, 2 ** 31 - 70):
        with pytest.raises(sa.SmolAttnError, match="rows"):
            sa.decode_shared(ctx, s.own.kv, s.slots[0], 0, s.own.kv, 1, None, [s.slots[1]], [far], q[:1], k[:1], v[:1], 4, 0.1)
    assert torch.equal(good, s.call(m, p))


# -------------------------------------------------------------------- evict

def evict_plain(mass, pos, n, end, keep, first, recent):
    """(dst, src, new mass, new positions) of one head, by the definition"""
    def rank(r):
        m = float(mass[r])
        if pos[r] < first or pos[r] >= end - recent:
            return (0, 0.0, r)
        return (1, 0.0, r) if m != m else (2, -m, r)

    order = sorted(range(n), key=rank)
    kept = set(order[:keep])
    left = min(n, keep)
    dst = [r for r in range(left) if r not in kept]
    src = [r for r in range(left, n) if r in kept]
    assert len(dst) == len(src)
    return dst, src


class Evict:
    def __init__(self, sa, ctx, hkv, hd, rows, keep, first=0, recent=0, seed=3, kind="random", extra=0):
        g = gen(seed)
        self.__dict__.update(sa=sa, hkv=hkv, hd=hd, rows=list(rows), keep=keep, first=first, recent=recent)
        n = len(rows)
        self.slots = [int(s) for s in torch.randperm(n + 1, generator=g)[:n]]
        self.own = Cache(sa, ctx, n + 1, hkv, hd, max(rows), g)
        stride = max(rows) + extra
        shape = (n + 1, hkv, stride)
        if kind == "random":
            self.mass = torch.exp(normal(g, *shape))
        elif kind == "ties":
            self.mass = torch.randint(0, 4, shape, generator=g).float() * 0.25
        elif kind == "equal":
            self.mass = torch.full(shape, 0.5)
        else:  # every kind of float
            self.mass = normal(g, *shape)
            pick = torch.randint(0, 12, shape, generator=g)
            for j, x in enumerate([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e-42, -1e-42]):
                self.mass[pick == j] = x
        self.pos = torch.argsort(torch.rand(shape, generator=g), -1).to(torch.int32)
        self.ends = [stride + 3 * i for i in range(n)]

    def call(self, apart):
        m, p = self.mass.cuda(), self.pos.cuda()
        mo, po = (torch.full_like(m, -7.0), torch.full_like(p, -7)) if apart else (None, None)
        return self.sa.kv_evict(self.own.kv, 1, self.slots, self.rows, self.ends, m, p, self.keep, first=self.first,
                                recent=self.recent, mass_out=mo, pos_out=po) + (m, p)

    def check(self, mo, po, m, p, apart):
        k, v = self.own.k.clone(), self.own.v.clone()
        wm = torch.full_like(self.mass, -7.0) if apart else self.mass.clone()
        wp = torch.full_like(self.pos, -7) if apart else self.pos.clone()
        moved = 0
        for n, s, end in zip(self.rows, self.slots, self.ends):
            left = min(n, self.keep)
            for h in range(self.hkv):
                dst, src = evict_plain(self.mass[s, h], self.pos[s, h], n, end, self.keep, self.first, self.recent)
                moved += len(dst)
                wm[s, h, :left], wp[s, h, :left] = self.mass[s, h, :left], self.pos[s, h, :left]
                for a, b in zip(dst, src):
                    wm[s, h, a], wp[s, h, a] = self.mass[s, h, b], self.pos[s, h, b]
                    k[s, h, a], v[s, h, a] = self.own.k[s, h, b], self.own.v[s, h, b]
        print("evict rows %s keep %d: %d moves" % (self.rows, self.keep, moved), flush=True)
        bits = lambda t: t.cpu().view(torch.int32)  # noqa: E731
        assert torch.equal(po.cpu(), wp)
        assert torch.equal(bits(mo), bits(wm))
        gk, gv = self.own.pull()
        assert torch.equal(gk.view(torch.int16), k.view(torch.int16))
        assert torch.equal(gv.view(torch.int16), v.view(torch.int16))
        if apart:
            assert torch.equal(bits(m), bits(self.mass)) and torch.equal(p.cpu(), self.pos)


@pytest.mark.parametrize("apart", [False, True], ids=["in_place", "apart"])
@pytest.mark.parametrize("c", [
    dict(hkv=2, hd=64, rows=[2], keep=1),
    dict(hkv=2, hd=64, rows=[0, 1, 40, 41], keep=40),
    dict(hkv=1, hd=72, rows=[300, 256, 257], keep=256, first=4, recent=32),
    dict(hkv=3, hd=80, rows=[1025, 1024, 999], keep=100, recent=100),
    dict(hkv=2, hd=128, rows=[2100, 2050], keep=2048, first=4, recent=512, extra=5),
    dict(hkv=1, hd=256, rows=[500], keep=499),
    dict(hkv=2, hd=96, rows=[500, 33], keep=120, kind="ties"),
    dict(hkv=2, hd=64, rows=[700], keep=350, kind="equal"),
    dict(hkv=2, hd=64, rows=[3000, 2000], keep=1000, kind="all", first=2, recent=10),
    dict(hkv=1, hd=64, rows=[70 + i for i in range(130)], keep=90),
], ids=lambda c: "%s-%d-%s" % ("_".join(map(str, c["rows"][:3])), c["keep"], c.get("kind", "random")))
def test_evict(sa, ctx, c, apart):
    e = Evict(sa, ctx, **c)
    e.check(*e.call(apart), apart)


@pytest.mark.parametrize("rows", [5000, 33000])
def test_evict_long(sa, ctx, rows):
    """more rows than the first and the second size of k_evict_select hold"""
    e = Evict(sa, ctx, 1, 64, [rows, rows - 1], rows // 3, recent=17, kind="ties")
    e.check(*e.call(False), False)


def test_evict_more_protected_than_kept(sa, ctx):
    """positions that a well-kept cache would not hold: still `keep` rows, the lowest protected ones"""
    e = Evict(sa, ctx, 2, 64, [100], 20, first=10, recent=10)
    e.pos[:] = 3
    e.check(*e.call(False), False)


def test_evict_refusals(sa, ctx):
    e = Evict(sa, ctx, 2, 64, [100, 50], 40)
    m, p = e.mass.cuda(), e.pos.cuda()
    mo, po = torch.empty_like(m), torch.empty_like(p)

    def refused(slots=e.slots, rows=e.rows, ends=e.ends, keep=40, mass=m, pos=p, **kw):
        with pytest.raises(sa.SmolAttnError):
            sa.kv_evict(e.own.kv, kw.pop("layer", 1), slots, rows, ends, mass, pos, keep, **kw)
    refused(layer=2)
    refused(layer=-1)
    refused(slots=[0, 0])
    refused(slots=[0, 3])
    refused(rows=[101, 50])
    refused(rows=[-1, 50])
    refused(rows=[100])
    refused(ends=[-1, 50])
    refused(keep=0)
    refused(first=41)
    refused(first=20, recent=21)
    refused(recent=2 ** 31 - 1)
    refused(first=-1)
    refused(mass=m[:, :, :99].contiguous(), pos=p[:, :, :99].contiguous())
    refused(mass_out=mo)
    refused(mass_out=m, pos_out=po)
    refused(mass_out=mo, pos_out=p)
    refused(mass_out=mo[:, :1].contiguous(), pos_out=po[:, :1].contiguous())
    ctx.synchronize()
    gk, gv = e.own.pull()
    assert torch.equal(gk.view(torch.int16), e.own.k.view(torch.int16))
    assert torch.equal(gv.view(torch.int16), e.own.v.view(torch.int16))


# ----------------------------------------------------------- together, graphs

def test_budgeted_stream(sa, ctx):
    """a stream held to a budget: scored steps, and an eviction whenever the rows reach it; every step against the
    definition on the rows that a plain program would have kept"""
    hq, hkv, hd, keep, most, steps = 4, 2, 64, 24, 32, 40
    g = gen(9)
    kv = sa.KVCache(ctx, 1, 1, hkv, hd, 64)
    rope = sa.RopeTable(ctx, hd, 1e4)
    mass = torch.zeros(1, hkv, 64, device="cuda")
    pos = torch.zeros(1, hkv, 64, dtype=torch.int32, device="cuda")
    rows, K, V, M, P = 0, [[] for _ in range(hkv)], [[] for _ in range(hkv)], [[] for _ in range(hkv)], [[] for _ in range(hkv)]
    for t in range(steps):
        q, k, v = normal(g, 1, hq * hd), normal(g, 1, hkv * hd), normal(g, 1, hkv * hd)
        out = sa.decode_scored(ctx, kv, 0, rope, [0], [rows], [t], q.cuda(), k.cuda(), v.cuda(), hq, hd ** -0.5, mass, pos)
        tab = table(sa, hd, 1e4, False, [t])
        q64, k64 = turned(q.view(1, hq, hd), None, tab, False)[0], turned(k.view(1, hkv, hd), None, tab, False)[0]
        v64 = v.double().view(hkv, hd)
        got = out.cpu().double().view(hkv, hq // hkv, hd)
        row_k, row_v = (torch.from_numpy(b.view(np.int16)).view(torch.bfloat16).double().view(hkv, hd)
                        for b in kv.read(0, 0, rows, 1))
        for h in range(hkv):
            kk = torch.stack(K[h] + [k64[h]])
            vv = torch.stack(V[h] + [v64[h]])
            o, p, pv, a = attend(q64.view(hkv, hq // hkv, hd)[h], kk, vv, hd ** -0.5, 0.0)
            assert ((got[h] - o).abs() <= 2 * err(hd, a) * pv + 2.0 ** -22 * o.abs()).all(), t
            for j, w in enumerate(p.sum(0).tolist()):
                if j < len(M[h]):
                    M[h][j] += w
                else:
                    M[h].append(w)
            # the row as the cache holds it (a 64-bit rotation may round to the next bf16)
            K[h].append(row_k[h])
            V[h].append(row_v[h])
            assert (row_k[h] - k64[h]).abs().max() <= 2.0 ** -8 * k64[h].norm()
            P[h].append(t)
        rows += 1
        if rows == most:
            sa.kv_evict(kv, 0, [0], [rows], [t + 1], mass, pos, keep, first=1, recent=8)
            for h in range(hkv):
                dst, src = evict_plain(M[h], P[h], rows, t + 1, keep, 1, 8)
                for a, b in zip(dst, src):
                    for x in (K, V, M, P):
                        x[h][a] = x[h][b]
                for x in (K, V, M, P):
                    del x[h][keep:]
            rows = keep
            assert pos.cpu()[0, :, :keep].tolist() == P
    ctx.synchronize()


def test_slots_past_32_bits(sa, ctx):
    """the last slots of a cache of more than 4 GB hold, give and lose the same rows as those of a small one"""
    hkv, hq, hd, rows, P = 8, 16, 128, 200, 300
    torch.manual_seed(4)
    K, V = (torch.randn(2, hkv, 320, hd, device="cuda").to(torch.bfloat16) for _ in range(2))
    q, k, v = (torch.randn(1, h * hd, device="cuda") for h in (hq, hkv, hkv))
    got = []
    for n_slots, cap in ((2, 320), (40, 65536)):
        kv = sa.KVCache(ctx, 1, n_slots, hkv, hd, cap)
        assert n_slots == 2 or n_slots * hkv * kv.capacity * hd * 2 > 2 ** 32
        kt, vt = kv.views(0)
        kt[-2:, :, :320] = K
        vt[-2:, :, :10] = V.view(2, hkv, 10, 32, hd).transpose(-1, -2)
        a, b = n_slots - 2, n_slots - 1
        out = [sa.decode_shared(ctx, kv, b, P, kv, 0, None, [a], [rows], q, k, v, hq, hd ** -0.5)]
        mass = torch.zeros(n_slots, hkv, 320, device="cuda")
        pos = torch.arange(320, dtype=torch.int32, device="cuda").expand(n_slots, hkv, 320).contiguous()
        out.append(sa.decode_scored(ctx, kv, 0, None, [b], [P], [P], q, k, v, hq, hd ** -0.5, mass, pos))
        sa.kv_evict(kv, 0, [b], [P + 1], [P + 1], mass, pos, 100, recent=10)
        out += [mass[b, :, :100].clone(), pos[b, :, :100].clone(), kt[-2:, :, :320].clone(), vt[-2:, :, :10].clone()]
        assert (kt[:-2].count_nonzero() + vt[:-2].count_nonzero()).item() == 0
        got.append(out)
        kv.close()
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_captured_steps_replay(sa):
    """a shared step, a scored step and an eviction in one graph, replayed with other inputs in the same buffers and
    eager work between the replays; growth under capture is refused"""
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        c2 = sa.Context(0)
        s = Shared(sa, c2, 4, 2, 64, [20, 33], 100)
        z = Scored(sa, c2, 4, 2, 64, [90, 70])
        m, p = z.arrays()
        mo, po = torch.zeros_like(m), torch.zeros_like(p)
        out_s, out_z = torch.empty(2, 256, device="cuda"), torch.empty(2, 256, device="cuda")

        def steps():
            s.call(out=out_s)
            z.call(m, p, out=out_z)
            sa.kv_evict(z.own.kv, 1, z.slots, [91, 71], [300, 300], m, p, 60, recent=4, mass_out=mo, pos_out=po)
        z.decay = 0.0
        steps()
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
            steps()
        for r in range(4):
            rg = gen(50 + r)
            s.dev[0][0].copy_(normal(rg, 2, 256))
            z.dev[0][0].copy_(normal(rg, 2, 256))
            z.own.push()
            torch.randn(1000, device="cuda").sum().item()
            g.replay()
            st.synchronize()
            got = [t.clone() for t in (out_s, out_z, m, mo, po)]
            rows = z.own.pull()
            z.own.push()
            steps()
            st.synchronize()
            for a, b in zip(got, (out_s, out_z, m, mo, po)):
                assert torch.equal(a.view(torch.int32), b.view(torch.int32)), r
            for a, b in zip(rows, z.own.pull()):
                assert torch.equal(a.view(torch.int16), b.view(torch.int16)), r
        big = Shared(sa, c2, 16, 8, 128, [100] * 20, 4000)
        big.dev = [t.cuda() for t in (big.q, big.k, big.v)], [big.qw.cuda(), big.kw.cuda()]
        st.synchronize()
        g2 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g2, stream=st, capture_error_mode="thread_local"):
            buf = torch.empty(20, 2048, device="cuda")
            with pytest.raises(sa.SmolAttnError, match="capture"):
                big.call(out=buf)
    st.synchronize()
    del s, z, big, g, g2
    c2.close()
