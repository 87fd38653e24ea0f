"""The projection with an adapter a row against its 64-bit form.

Bounds, derived before any run. The shared product is an fp32 sum of exact
products, x carried to 2^-16 on smol_linear_dev's GEMM path (two bf16 parts),
so (2 (in + 1) 2^-24 + 2^-16) sum |x w| + 2^-22 |bias|. The low-rank part carries
x and t whole (three bf16 parts): t is off by at most 2 (in + 20) 2^-24 sum |a x|
(20: the chunks' and the waves' partial sums), and B t by that through |B| and
2 (rank + 2) 2^-24 sum |b| |t|. A bf16 y is truncated: one step, 2^-7 of the
value, more.
"""
import numpy as np
import pytest

from conftest import pkg  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


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


class Case:
    def __init__(self, seq, k, n, ranks, bf16=False, bias=True, ids=None, seed=1, bare=0.1):
        g = torch.Generator()
        g.manual_seed(seed)
        rn = lambda *s: torch.randn(s, generator=g)  # noqa: E731
        self.x = rn(seq, k).to(torch.bfloat16 if bf16 else torch.float32)
        self.w = (rn(n, k) * k ** -0.5).to(torch.bfloat16)
        self.bias = rn(n) if bias else None
        self.ab = [((rn(r, k) * k ** -0.5).to(torch.bfloat16), (rn(n, r) * r ** -0.5).to(torch.bfloat16), 0.25 + 0.5 * i)
                   for i, r in enumerate(ranks)]
        if ids is None:
            ids = torch.randint(0, len(ranks), (seq,), generator=g)
            ids[torch.rand(seq, generator=g) < bare] = -1
            ids = ids.tolist()
        self.ids, self.bf16 = ids, bf16

    def exact(self):
        """y and its bound in 64 bits"""
        x, w = self.x.double(), self.w.double()
        k = w.shape[1]
        y, b = x @ w.T, x.abs() @ w.abs().T * (2 * (k + 1) * 2.0 ** -24 + 2.0 ** -16)
        if self.bias is not None:
            y, b = y + self.bias.double(), b + 2.0 ** -22 * self.bias.abs().double()
        for s, i in enumerate(self.ids):
            if i < 0:
                continue
            a, bb, scale = self.ab[i][0].double(), self.ab[i][1].double(), self.ab[i][2]
            t = a @ x[s]
            te = 2 * (k + 20) * 2.0 ** -24 * (a.abs() @ x[s].abs())
            y[s] += scale * (bb @ t)
            b[s] += scale * (bb.abs() @ (te + 2 * (len(t) + 2) * 2.0 ** -24 * t.abs()))
        return y, b + 2.0 ** -23 * y.abs()

    def to(self, sa, ctx):
        self.set = sa.Adapters(ctx, [(a.cuda(), b.cuda(), s) for a, b, s in self.ab])
        self.dev = self.x.cuda(), self.w.cuda(), None if self.bias is None else self.bias.cuda()

    def call(self, sa, ctx, out_bf16=False, **kw):
        if not hasattr(self, "set"):
            self.to(sa, ctx)
        x, w, bias = self.dev
        return sa.linear_adapters(ctx, x, w, self.set, self.ids, bias=bias, out_bf16=out_bf16, **kw)

    def check(self, y, out_bf16=False):
        want, tol = self.exact()
        got = (y.view(torch.bfloat16) if out_bf16 else y).cpu().double()
        if out_bf16:
            tol = tol + 2.0 ** -7 * want.abs()
        worst = float(((got - want).abs() / tol).max())
        print("adapters %s ranks %s: %.3f of the bound" % (tuple(want.shape), [len(a[0]) for a in self.ab][:6], worst), flush=True)
        assert worst <= 1.0


CASES = [
    dict(seq=1, k=64, n=64, ranks=[8]),
    dict(seq=1, k=1, n=1, ranks=[1]),
    dict(seq=3, k=1024, n=512, ranks=[8, 16, 1]),
    dict(seq=4, k=37, n=70, ranks=[3, 5]),
    dict(seq=5, k=1021, n=333, ranks=[4, 17, 33]),
    dict(seq=16, k=256, n=130, ranks=[64, 128]),
    dict(seq=17, k=640, n=1000, ranks=[16]),
    dict(seq=40, k=520, n=256, ranks=[8] * 40, bare=0.5),
    dict(seq=33, k=72, n=129, ranks=[100, 2, 31, 32], bias=False),
    dict(seq=300, k=512, n=768, ranks=[16, 32, 48]),
    dict(seq=700, k=136, n=64, ranks=[8] * 60),
    # the last rows of the one-launch form and the first past it, an in_dim that needs padded copies
    dict(seq=32, k=2048, n=48, ranks=[16, 4]),
    dict(seq=64, k=96, n=200, ranks=[20] * 50),
    dict(seq=65, k=97, n=90, ranks=[12, 40]),
    # few rows and ranks, one launch: four tiles of ranks, a set whose largest rank no row uses, the last sizes and the next
    dict(seq=16, k=256, n=100, ranks=[17, 20]),
    dict(seq=5, k=333, n=65, ranks=[64]),
    dict(seq=4, k=1000, n=48, ranks=[16, 16, 16, 16], ids=[3, 1, 0, 2]),
    dict(seq=3, k=96, n=40, ranks=[128, 8, 33], ids=[2, -1, 1]),
    dict(seq=16, k=1024, n=33, ranks=[16], bare=0.0),
    dict(seq=16, k=1032, n=33, ranks=[16], bare=0.0),
    dict(seq=200, k=333, n=1001, ranks=[128, 8]),
]


@pytest.mark.parametrize("out_bf16", [False, True], ids=["f32", "y_bf16"])
@pytest.mark.parametrize("bf16", [False, True], ids=["x_f32", "x_bf16"])
@pytest.mark.parametrize("c", CASES, ids=lambda c: "%d-%d-%d-%s" % (c["seq"], c["k"], c["n"], c["ranks"][:2]))
def test_adapters(sa, ctx, c, bf16, out_bf16):
    t = Case(bf16=bf16, **c)
    t.check(t.call(sa, ctx, out_bf16), out_bf16)


def test_no_row_has_one(sa, ctx):
    """the shared product alone, bit for bit smol_linear_dev's"""
    t = Case(9, 128, 96, [8], ids=[-1] * 9)
    y = t.call(sa, ctx)
    assert torch.equal(y, sa.linear(ctx, t.dev[0], t.dev[1], t.dev[2]))


@pytest.mark.parametrize("seq,k,n", [(65, 64, 48), (130, 96, 257), (1000, 72, 300)])
def test_bare_rows_among_others(sa, ctx, seq, k, n):
    """a bf16 y of many rows: those without an adapter are smol_linear_dev's bits, whatever the adapters hold"""
    t = Case(seq, k, n, [8, 16], bf16=True, bare=0.4)
    y = t.call(sa, ctx, True)
    t.check(y, True)
    z = sa.linear(ctx, t.dev[0], t.dev[1], t.dev[2], out_bf16=True)
    bare = [s for s in range(seq) if t.ids[s] < 0]
    assert bare and torch.equal(y[bare], z[bare])
    for a, b, _ in t.ab:
        a.fill_(float("nan"))
        b.fill_(float("inf"))
    t.to(sa, ctx)
    assert torch.equal(t.call(sa, ctx, True)[bare], z[bare])


@pytest.mark.parametrize("n", [9, 50, 130])
def test_rows_do_not_meet(sa, ctx, n):
    """a NaN row, and NaN weights of an adapter, reach their own rows only"""
    t = Case(n, 256, 192, [8, 16, 24])
    t.ids = [i % 4 - 1 for i in range(n)]
    clean = t.call(sa, ctx).clone()
    t.check(clean)
    t.ab[1][0][3] = float("nan")
    t.to(sa, ctx)
    t.dev[0][6] = float("nan")
    y = t.call(sa, ctx)
    hit = [s for s in range(n) if t.ids[s] == 1 or s == 6]
    rest = [s for s in range(n) if s not in hit]
    assert torch.isnan(y[hit]).all() and torch.equal(y[rest], clean[rest])


@pytest.mark.parametrize("n", [8, 32, 64, 128])
def test_a_row_does_not_depend_on_the_order(sa, ctx, n):
    """the same rows in another order, with the same number of rows an adapter: the same bits a row"""
    t = Case(n, 512, 256, [16, 8])
    t.ids = [s % 2 for s in range(n)]
    y = t.call(sa, ctx).clone()
    perm = torch.arange(n - 1, -1, -1)
    t.dev = (t.dev[0][perm.cuda()].contiguous(),) + t.dev[1:]
    t.ids = [t.ids[int(i)] for i in perm]
    assert torch.equal(t.call(sa, ctx), y[perm.cuda()])


def test_captured(sa):
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        c2 = sa.Context(0)
        t = Case(20, 256, 192, [8, 16])
        out = torch.empty(20, 192, device="cuda")
        t.call(sa, c2, out=out)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
            t.call(sa, c2, out=out)
        for r in range(4):
            t.dev[0].normal_()
            torch.randn(1000, device="cuda").sum().item()
            g.replay()
            st.synchronize()
            got = out.clone()
            t.call(sa, c2, out=out)
            st.synchronize()
            assert torch.equal(got, out)
        many = Case(700, 64, 64, [8] * 60)
        many.to(sa, c2)
        big = torch.empty(700, 64, device="cuda")
        st.synchronize()
        g2 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g2, stream=st, capture_error_mode="thread_local"):
            with pytest.raises(sa.SmolAttnError, match="capture"):
                many.call(sa, c2, out=big)
    st.synchronize()
    del t, many, g, g2
    c2.close()


def test_refusals(sa, ctx):
    t = Case(6, 64, 48, [8, 4])
    y = t.call(sa, ctx).clone()
    x, w, bias = t.dev
    bad = lambda **k: pytest.raises(sa.SmolAttnError)  # noqa: E731
    for ids in ([0] * 5, [0] * 5 + [2], [0] * 5 + [-2]):
        with bad():
            sa.linear_adapters(ctx, x, w, t.set, ids, bias=bias)
    for args in ((x[:, :32].contiguous(), w), (x, w[:40]), (x.double(), w), (x, w.float()), (x.t().contiguous().t(), w)):
        with bad():
            sa.linear_adapters(ctx, args[0], args[1], t.set, t.ids)
    with bad():
        sa.linear_adapters(ctx, x, w, t.set, t.ids, bias=bias[:40])
    with bad():
        sa.linear_adapters(ctx, x, w, t.set, t.ids, out=torch.empty(6, 47, device="cuda"))
    a, b = t.ab[0][0].cuda(), t.ab[0][1].cuda()
    for ab in ([], [(a, b[:, :7].contiguous(), 1.0)], [(a[:0], b[:, :0].contiguous(), 1.0)], [(a.float(), b, 1.0)],
               [(torch.zeros(129, 64, dtype=torch.bfloat16, device="cuda"),
                 torch.zeros(48, 129, dtype=torch.bfloat16, device="cuda"), 1.0)]):
        with bad():
            sa.Adapters(ctx, ab)
    c2 = sa.Context(0)
    with bad():
        sa.linear_adapters(c2, x, w, t.set, t.ids)
    c2.close()
    one = torch.zeros(2000, device="cuda")
    import ctypes
    ids = np.zeros(6, np.int32)
    rc = sa.load().smol_linear_adapters_dev(ctx.h, one.data_ptr(), 0, one.data_ptr() + 16, 0, w.data_ptr(), None, 6, 64, 48,
                                            t.set.h, ids.ctypes.data_as(ctypes.POINTER(ctypes.c_int)))
    assert rc == -1
    assert torch.equal(t.call(sa, ctx), y)
    # y over the weights
    wy = torch.zeros(48 * 64 + 6 * 48, dtype=torch.float32, device="cuda")
    rc = sa.load().smol_linear_adapters_dev(ctx.h, wy.data_ptr(), 0, x.data_ptr(), 0, wy.data_ptr() + 256, None, 6, 64, 48,
                                            t.set.h, ids.ctypes.data_as(ctypes.POINTER(ctypes.c_int)))
    assert rc == -1
    assert torch.equal(y, t.call(sa, ctx))


def test_captured_runs(sa):
    """prompts one after the other: more tiles than the arguments' table holds, captured as runs"""
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        c2 = sa.Context(0)
        t = Case(180, 64, 80, [8] * 60, ids=[s // 3 for s in range(180)])
        out = torch.empty(180, 80, device="cuda")
        t.call(sa, c2, out=out)
        st.synchronize()
        t.check(out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
            t.call(sa, c2, out=out)
        for r in range(3):
            t.dev[0].normal_()
            g.replay()
            st.synchronize()
            got = out.clone()
            t.call(sa, c2, out=out)
            st.synchronize()
            assert torch.equal(got, out)
    st.synchronize()
    del t, g
    c2.close()


def test_serving_steps(sa, ctx):
    """decode steps of a batch whose requests share a prompt and have adapters of their own: the projections' outputs are the
    attention's inputs and its output the last projection's; every stage against its 64-bit form on the inputs it got"""
    from test_gpu_shared import attend, err, table, turned
    n, dim, hq, hkv, hd, P = 5, 192, 8, 4, 64, 70
    ids = [2, -1, 0, 2, 1]
    cases = [Case(n, dim, h * hd, [8, 16, 4], ids=ids, bias=b, seed=10 + i)
             for i, (h, b) in enumerate(((hq, True), (hkv, True), (hkv, False)))]
    last = Case(n, hq * hd, dim, [8, 16, 4], ids=ids, bias=False, seed=20)
    for t in cases + [last]:
        t.to(sa, ctx)
    pre, kv = sa.KVCache(ctx, 1, 1, hkv, hd, 128), sa.KVCache(ctx, 1, n, hkv, hd, 64)
    kt, vt = pre.views(0)
    torch.manual_seed(3)
    kt.normal_()
    vt.normal_()
    pk, pv = kt[0].cpu().double(), vt[0].transpose(-1, -2).reshape(hkv, -1, hd).cpu().double()
    rope = sa.RopeTable(ctx, hd, 1e4)
    lens = [0] * n
    own = [[] for _ in range(n)]
    for step in range(3):
        x = torch.randn(n, dim)
        for t in cases:
            t.x = x
            t.dev = (x.cuda(),) + t.dev[1:]
        q, k, v = (t.call(sa, ctx) for t in cases)
        for t, y in zip(cases, (q, k, v)):
            t.check(y)
        att = sa.decode_shared(ctx, pre, 0, P, kv, 0, rope, list(range(n)), lens, q, k, v, hq, hd ** -0.5)
        rows = table(sa, hd, 1e4, False, [P + l for l in lens])
        q64 = turned(q.cpu().view(n, hq, hd), None, rows, False).view(n, hkv, hq // hkv, hd)
        k64 = turned(k.cpu().view(n, hkv, hd), None, rows, False)
        v64 = v.cpu().double().view(n, hkv, hd)
        got = att.cpu().double().view(n, hkv, hq // hkv, hd)
        for i in range(n):
            for h in range(hkv):
                kk = torch.cat([pk[h, :P]] + [r[0][h:h + 1] for r in own[i]] + [k64[i, h:h + 1]])
                vv = torch.cat([pv[h, :P]] + [r[1][h:h + 1] for r in own[i]] + [v64[i, h:h + 1]])
                o, _, w, a = attend(q64[i, h], kk, vv, hd ** -0.5, 0.0)
                assert ((got[i, h] - o).abs() <= 2 * err(hd, a) * w + 2.0 ** -22 * o.abs()).all(), (step, i, h)
            # the rows as the cache holds them
            rk, rv = (torch.from_numpy(b.view(np.int16)).view(torch.bfloat16).double().view(hkv, hd)
                      for b in kv.read(0, i, lens[i], 1))
            own[i].append((rk, rv))
        last.x = att.cpu()
        last.dev = (att,) + last.dev[1:]
        last.check(last.call(sa, ctx))
        lens = [l + 1 for l in lens]
    pre.close()
    kv.close()
