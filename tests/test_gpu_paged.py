"""A KV cache in pages against plain 64-bit forms: rows in and back, the decode step over all rows and over chosen pages.

Bounds, derived before any run. Half a step of a rounding: fp32 2^-24, bf16 2^-8 of the value.
Rows. The norm and the rotation take about eight fp32 roundings of terms of a pair: 2^-20 of the row's norm covers them.
bf16 rows: 2^-8 |x| + that. Codes: s is within 2^-20 of amax / 127 (norm and rotation of the largest element, two roundings), a
value within s / 2 of x, plus what x itself is off by and the two roundings of x * (127 / amax): 127 s 2^-20 more.
Scores. Q is carried at 2^-24 of its row's largest element (24-bit numbers) or whole (three bf16 parts), and its norm, rotation
and scaling are eight roundings, the fp32 sum of bf16 products hd: |ds| <= (hd + 16) 2^-24 a with
a = max_j scale sum_d max|q| |k_jd|. Weights: e = 2 (hd + 16) 2^-24 a + 2^-20 (exp, sums, joins; bf16 parts leave 2^-24).
Codes' weights are 24-bit numbers against the largest p s of their 64 rows: each is off by 2^-24 of it at most, times 127:
sum over the units of 64 127 2^-24 max(p s), with p normalised.
out: 2 e sum_j p_j |v_j| + that + 2^-22 |exact|.
"""
import math

import numpy as np
import pytest

from conftest import pkg  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

EPS = 1e-6
P = 64


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


def order(codes):
    r = np.arange(P)
    t, g, i = r // 16, r % 16 // 4, r % 4
    return torch.from_numpy(g * 16 + t * 4 + i if codes else t // 2 * 32 + g * 8 + t % 2 * 4 + i)


def normal(g, *shape, bf16=False, std=1.0):
    x = torch.randn(shape, generator=g) * std
    return x.to(torch.bfloat16) if bf16 else x


def i32(a):
    return torch.as_tensor(a, dtype=torch.int32).cuda()


def outward(x, up):
    """fp32 as the next bf16 at or above (below)"""
    b = x.to(torch.bfloat16).float()
    wrong = b < x if up else b > x
    # the other neighbour: bf16 numbers are those with the low 16 bits zero
    bits = x.view(torch.int32) & -65536
    cut = bits.view(torch.float32)
    away = (bits + 65536).view(torch.float32)
    other = torch.where((x > 0) == up, away, cut)
    return torch.where(wrong, other, b)


class Pool:
    """a pool on the device whose pages all hold something, and its contents on the host"""

    def __init__(self, sa, ctx, n_pages, hkv, hd, codes, g, layers=2, layer=1, spread=1.0):
        self.sa, self.ctx, self.hkv, self.hd, self.codes, self.layer, self.n = sa, ctx, hkv, hd, codes, layer, n_pages
        self.pool = sa.KVPages(ctx, layers, n_pages, hkv, hd, sa.INT8 if codes else sa.BF16)
        k, v, s, b = self.views = self.pool.views(layer)
        kk = normal(g, n_pages, hkv, P, hd) * spread
        vv = normal(g, n_pages, hkv, P, hd)
        e = 16 if codes else 8
        pad = -hd % e
        if codes:
            sc = torch.exp(normal(g, n_pages, hkv, 2, P, std=0.2)) / 42
            kk, vv = ((x / sc[:, :, i, :, None]).round().clamp(-127, 127) for i, x in enumerate((kk, vv)))
            s.copy_(sc)
            stored = kk * sc[:, :, 0, :, None]
        else:
            kk, vv = kk.to(torch.bfloat16).float(), vv.to(torch.bfloat16).float()
            stored = kk
        k.copy_(torch.nn.functional.pad(kk, (0, pad)).view(n_pages, hkv, P, -1, e).transpose(2, 3))
        line = torch.empty(n_pages, hkv, hd, P)
        line[..., order(codes)] = vv.transpose(2, 3)
        v.copy_(line if codes else line.view(n_pages, hkv, hd, 2, 32).transpose(2, 3))
        b.copy_(torch.stack([outward(stored.amin(2), False), outward(stored.amax(2), True)], 2))

    def bits(self):
        """the layer's arrays as whole numbers, to see what changed"""
        return [None if x is None else x.cpu().view({1: torch.int8, 2: torch.int16, 4: torch.int32}[x.element_size()]).clone()
                for x in self.views]

    def rows(self):
        """K and V [pages, kv, 64, hd] as the values they stand for, 64 bits"""
        k, v, s, _ = (None if x is None else x.cpu() for x in self.views)
        k = k.double().transpose(2, 3).flatten(3)[..., :self.hd]
        v = v.double()
        if not self.codes:
            v = v.transpose(2, 3).flatten(3)
        v = v[..., order(self.codes)].transpose(2, 3)
        if self.codes:
            k, v = k * s[:, :, 0, :, None].double(), v * s[:, :, 1, :, None].double()
        return k, v


def table_of(g, n_pages, needs, stride=None, bad=-7):
    """pages for every sequence, in no order; entries that nobody may look at are none"""
    stride = stride or max(max(needs), 1) + 1
    perm = torch.randperm(n_pages, generator=g)
    t = torch.full((len(needs), stride), bad, dtype=torch.int32)
    at = 0
    for i, m in enumerate(needs):
        t[i, :m] = perm[at:at + m]
        at += m
    return t


def angles(sa, hd, theta, inter, pos):
    c, s = zip(*(sa.rope_fill_host(int(p), 1, hd, theta, 1 if inter else 0) for p in pos))
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


def check_stored(pool, before, wrote, k64, v64):
    """rows (page, row, index into k64 / v64) are what the formulas make of k64, v64 [m, kv, hd], their pages' bounds hold them,
    and nothing else changed. before: the layer's bits"""
    after = pool.bits()
    kv, vv = pool.rows()
    codes, hd = pool.codes, pool.hd
    o = order(codes)
    expect = [x if x is None else x.clone() for x in before]
    for page, row, m in wrote:
        for x64, got, is_k in ((k64[m], kv[page, :, row], True), (v64[m], vv[page, :, row], False)):
            norm = x64.norm(dim=-1, keepdim=True) if is_k else 0 * x64[..., :1]
            off = 2.0 ** -20 * norm
            if codes:
                amax = x64.abs().amax(-1, keepdim=True)
                s = pool.views[2][page, :, 0 if is_k else 1, row].cpu().double()[:, None]
                assert ((s - amax / 127).abs() <= off / 127 + 2.0 ** -22 * amax / 127).all()
                assert ((got - x64).abs() <= s / 2 + off + 127 * s * 2.0 ** -20).all()
            else:
                assert ((got - x64).abs() <= 2.0 ** -8 * x64.abs() + off).all()
        a = int(o[row])
        expect[0][page, :, :, row] = after[0][page, :, :, row]
        if codes:
            expect[1][page, :, :, a] = after[1][page, :, :, a]
            expect[2][page, :, :, row] = after[2][page, :, :, row]
        else:
            expect[1][page, :, a // 32, :, a % 32] = after[1][page, :, a // 32, :, a % 32]
    old = before[3].view(torch.bfloat16).float()
    for page in {w[0] for w in wrote}:
        rows = [w[1] for w in wrote if w[0] == page]
        x = kv[page, :, rows].float()  # products of a code and its scale, rounded as the kernel rounds them
        lo, hi = x.amin(1), x.amax(1)
        if 0 not in rows:
            lo, hi = torch.minimum(lo, old[page, :, 0]), torch.maximum(hi, old[page, :, 1])
        b = torch.stack([outward(lo, False), outward(hi, True)], 1)
        assert torch.equal(b, after[3][page].view(torch.bfloat16).float()), page
        expect[3][page] = after[3][page]
    if codes and hd % 16:
        pad = pool.views[0][:, :, -1, :, hd % 16:].cpu()
        for page, row, _ in wrote:
            assert (pad[page, :, row] == 0).all()
    for e, x in zip(expect, after):
        assert e is None or torch.equal(e, x)


# ------------------------------------------------------------------ rows in and back

HEADS = [(2, 64, False), (1, 72, True), (5, 80, False), (2, 96, True), (8, 128, False), (1, 256, True)]


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("hkv,hd,inter", HEADS)
@pytest.mark.parametrize("bf16,norm,rope", [(False, True, True), (True, False, True), (False, True, False)])
def test_append_and_read(sa, ctx, hkv, hd, inter, codes, bf16, norm, rope):
    g = torch.Generator().manual_seed(hd * 8 + codes)
    lens = [1, 64, 0, 65, 130, 17, 3]
    pos = [0, 64, 5, 63, 1, 100, 62]
    needs = [-(-(p + l) // P) for p, l in zip(pos, lens)]
    pool = Pool(sa, ctx, sum(needs) + 3, hkv, hd, codes, g)
    t = table_of(g, pool.n, needs)
    for i, (p, l) in enumerate(zip(pos, lens)):  # pages that no row of the call is in need not exist
        t[i, :p // P if l else needs[i]] = -1
    rows = sum(lens)
    k, v = normal(g, rows, hkv * hd, bf16=bf16), normal(g, rows, hkv * hd, bf16=bf16)
    w = 1.0 + 0.2 * normal(g, hd) if norm else None
    table = sa.RopeTable(ctx, hd, 1e4, 1 if inter else 0) if rope else None
    starts = [0]
    for l in lens:
        starts.append(starts[-1] + l)
    where = [(i, p + r) for i, (p, l) in enumerate(zip(pos, lens)) for r in range(l)]
    k64 = turned(k.view(rows, hkv, hd), w, angles(sa, hd, 1e4, inter, [x for _, x in where]) if rope else None, inter)
    v64 = v.double().view(rows, hkv, hd)
    before = pool.bits()
    td, sd, pd = t.cuda(), i32(starts), i32(pos)
    print("append hkv %d hd %d codes %d" % (hkv, hd, codes), flush=True)
    sa.pages_append(pool.pool, pool.layer, table, td, sd, pd, k.cuda(), v.cuda(), k_norm=None if w is None else w.cuda(), eps=EPS)
    ctx.synchronize()
    check_stored(pool, before, [(int(t[i, x // P]), x % P, m) for m, (i, x) in enumerate(where)], k64, v64)
    if codes and not bf16:
        # V goes in as it is: its codes and scales are the formula's to the last bit
        top = v.view(rows, hkv, hd).abs().amax(-1, keepdim=True)
        want = torch.round(v.view(rows, hkv, hd) * (torch.tensor(127.0) / top))
        got = pool.views[1].cpu()[..., order(True)].transpose(2, 3)
        sc = pool.views[2].cpu()
        for m, (i, x) in enumerate(where):
            assert torch.equal(got[int(t[i, x // P]), :, x % P].float(), want[m])
            assert torch.equal(sc[int(t[i, x // P]), :, 1, x % P], (top / 127.0)[m, :, 0])
    kk, vv = pool.rows()
    want = [torch.stack([x[int(t[i, p // P]), :, p % P] for i, p in where]).flatten(1) for x in (kk, vv)]
    for dtype in (torch.float32, torch.bfloat16):
        print("read", dtype, flush=True)
        a, b = sa.pages_read(pool.pool, pool.layer, td, sd, pd, rows, dtype=dtype)
        ctx.synchronize()
        for x, y in ((a, want[0]), (b, want[1])):
            assert torch.equal(x.cpu(), y.float().to(dtype))


def test_rows_of_codes_at_the_ends(sa, ctx):
    """rows of zeros, tiny and huge rows, rows with a NaN or an infinity: as values, and the bounds they leave"""
    g = torch.Generator().manual_seed(5)
    hkv, hd = 2, 128
    pool = Pool(sa, ctx, 3, hkv, hd, True, g)
    x = normal(g, 8, hkv, hd)
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 2.0 ** -88
    x[3] *= 1e30
    x[4, 0, 7] = math.nan
    x[5, 1, 3] = -math.inf
    x[6, 0] = 0
    x[6, 0, 5] = math.inf
    t, starts, pos = torch.tensor([[2]], dtype=torch.int32).cuda(), i32([0, 8]), i32([0])
    k = x.view(8, -1).cuda()
    sa.pages_append(pool.pool, 1, None, t, starts, pos, k, k.clone())
    a, b = sa.pages_read(pool.pool, 1, t, starts, pos, 8, dtype=torch.float32)
    ctx.synchronize()
    for got in (a.cpu().view(8, hkv, hd), b.cpu().view(8, hkv, hd)):
        assert (got[0] == 0).all() and (got[1] == 0).all()
        for m in (2, 3, 7):
            s = x[m].abs().amax(-1, keepdim=True) / 127
            assert ((got[m] - x[m]).abs() <= s * (0.5 + 127 * 2.0 ** -20)).all()
        for m, h in ((4, 0), (5, 1), (6, 0)):
            assert got[m, h].isnan().all() and got[m, 1 - h].isfinite().all()
    assert pool.views[3][2].isnan().all()
    # a new first row starts the page's bounds anew
    sa.pages_append(pool.pool, 1, None, t, i32([0, 1]), pos, k[7:], k[7:].clone())
    ctx.synchronize()
    bounds = pool.views[3][2].float().cpu()
    assert bounds.isfinite().all() and (bounds[:, 0] <= bounds[:, 1]).all()


# ------------------------------------------------------------------ decode

def attend(q, k, v, scale, cap, codes, hd, unit_of):
    """q [G, hd], k, v [m, hd] in 64 bits: out and its bound; unit_of: the unit that row j of them is quantised with"""
    z = q @ k.T * scale
    if cap:
        z = cap * torch.tanh(z / cap)
    p = torch.softmax(z, -1)
    a = float((q.abs().amax(-1, keepdim=True) * k.abs().sum(-1)).max() * scale)
    e = 2 * (hd + 16) * 2.0 ** -24 * a + 2.0 ** -20
    o = p @ v
    tol = 2 * e * (p @ v.abs()) + 2.0 ** -22 * o.abs()
    if codes:
        top = p * v.abs().amax(-1)
        for u in unit_of.unique():
            tol = tol + 64 * 2.0 ** -24 * top[:, unit_of == u].amax(-1, keepdim=True) * 2  # amax may be half of 127 s
    return o, tol


class Step:
    """one decode step's inputs, its call and its check"""

    def __init__(self, sa, ctx, hq, hkv, hd, lens, codes, inter=False, norm=True, bf16=False, window=0, cap=0.0, rope=True, seed=1,
                 std=1.0, top=0, first=1, recent=1, stride=None, spread=1.0, shared=0):
        g = torch.Generator().manual_seed(seed)
        self.__dict__.update(sa=sa, ctx=ctx, hq=hq, hkv=hkv, hd=hd, lens=list(lens), codes=codes, inter=inter, window=window, cap=cap,
                             top=top, first=first, recent=recent)
        n = self.n = len(self.lens)
        needs = [l // P + 1 if l >= 0 else 0 for l in self.lens]
        self.pool = Pool(sa, ctx, sum(needs) + 2, hkv, hd, codes, g, spread=spread)
        self.t = table_of(g, self.pool.n, needs, stride)
        if window:
            for i, l in enumerate(self.lens):  # pages before the window need not exist
                self.t[i, :max(0, l - window + 1) // P] = -1
        for i in range(1, n if shared else 1):  # a common prefix
            m = min(shared, needs[0] - 1, needs[i] - 1)
            self.t[i, :m] = self.t[0, :m]
        self.q = normal(g, n, hq * hd, bf16=bf16, std=std)
        self.k = normal(g, n, hkv * hd, bf16=bf16)
        self.v = normal(g, n, hkv * hd, bf16=bf16)
        self.qw = 1.5 + 0.1 * normal(g, hd) if norm else None
        self.kw = 1.0 + 0.1 * normal(g, hd) if norm else None
        self.rope = sa.RopeTable(ctx, hd, 1e4, 1 if inter else 0) if rope else None
        self.scale = hd ** -0.5
        d = lambda x: None if x is None else x.cuda()  # noqa: E731
        self.dev = dict(q=d(self.q), k_new=d(self.k), v_new=d(self.v)), dict(q_norm=d(self.qw), k_norm=d(self.kw))
        self.td, self.ld = self.t.cuda(), i32(self.lens)
        self.before = self.pool.bits()
        self.rows = self.pool.rows()

    def call(self, **kw):
        a, b = self.dev
        if self.top:
            out, self.chosen = self.sa.decode_paged_top(
                self.ctx, self.pool.pool, self.pool.layer, self.rope, self.td, self.ld, a["q"], a["k_new"], a["v_new"], self.hq,
                self.scale, self.top, first=self.first, recent=self.recent, cap=self.cap, eps=EPS, **b, **kw)
            return out
        return self.sa.decode_paged(self.ctx, self.pool.pool, self.pool.layer, self.rope, self.td, self.ld, a["q"], a["k_new"],
                                    a["v_new"], self.hq, self.scale, window=self.window, cap=self.cap, eps=EPS, **b, **kw)

    def turned(self):
        n, hd = self.n, self.hd
        rope = angles(self.sa, hd, 1e4, self.inter, [max(l, 0) for l in self.lens]) if self.rope else None
        return (turned(self.q.view(n, self.hq, hd), self.qw, rope, self.inter),
                turned(self.k.view(n, self.hkv, hd), self.kw, rope, self.inter), self.v.double().view(n, self.hkv, hd))

    def choose(self, i, h, q):
        """the pages of (sequence, kv head) that the formula chooses"""
        pages = -(-self.lens[i] // P)
        if pages <= self.top:
            return list(range(pages))
        b = self.before[3].view(torch.bfloat16)[self.t[i, :pages].long(), h].double()  # [pages, 2, hd]
        score = torch.zeros(pages, dtype=torch.float64)
        for x in q * self.scale:
            score += torch.maximum(b[:, 0] * x, b[:, 1] * x).sum(-1)
        rank = [(0 if j < self.first or j >= pages - self.recent else 1 if math.isnan(s) else 2, -s if s == s else 0, j)
                for j, s in enumerate(score.tolist())]
        return sorted(j for _, _, j in sorted(rank)[:self.top])

    def check(self, out, stored=True, what=""):
        q, k, v = self.turned()
        G, hd = self.hq // self.hkv, self.hd
        out = out.cpu().double().view(self.n, self.hkv, G, hd)
        kk, vv = self.rows
        worst = 0.0
        for i, l in enumerate(self.lens):
            if l < 0:
                continue
            lo = max(0, l - self.window + 1) if self.window else 0
            for h in range(self.hkv):
                qh = q[i].view(self.hkv, G, hd)[h]
                at = torch.arange(lo, l)
                if self.top:
                    pages = self.choose(i, h, qh)
                    got = self.chosen[i, h].tolist()
                    assert got == pages + [-1] * (self.top - len(pages)), (i, h, got, pages)
                    at = at[torch.isin(at // P, torch.tensor(pages, dtype=torch.long))]
                page = self.t[i, at // P].long()
                keys = torch.cat([kk[page, h, at % P], k[i, h:h + 1]])
                vals = torch.cat([vv[page, h, at % P], v[i, h:h + 1]])
                o, tol = attend(qh, keys, vals, self.scale, self.cap, self.codes, hd, torch.cat([at // P, torch.tensor([1 << 30])]))
                assert torch.isfinite(out[i, h]).all(), (i, h)
                worst = max(worst, float(((out[i, h] - o).abs() / tol).max()))
        print("paged%s hq %d hkv %d hd %d codes %d lens %s: %.3f of the bound" % (what, self.hq, self.hkv, hd, self.codes,
                                                                               self.lens[:6], worst), flush=True)
        assert worst <= 1.0
        if stored:
            live = [i for i in range(self.n) if self.lens[i] >= 0]
            check_stored(self.pool, self.before, [(int(self.t[i, self.lens[i] // P]), self.lens[i] % P, i) for i in live], k, v)


DECODE = [
    dict(hq=4, hkv=2, hd=64, lens=[0]),
    dict(hq=4, hkv=2, hd=64, lens=[1]),
    dict(hq=2, hkv=2, hd=72, lens=[0, 1, 31, 32, 33], inter=True),
    dict(hq=15, hkv=5, hd=80, lens=[63, 64, 65], norm=False),
    dict(hq=6, hkv=1, hd=96, lens=[100, 0, 7, 128], bf16=True),
    dict(hq=16, hkv=8, hd=128, lens=[500, 3, 1024, 129]),
    dict(hq=8, hkv=1, hd=256, lens=[300, 1, 700], inter=True, cap=30.0),
    dict(hq=8, hkv=4, hd=256, lens=[64, 4], inter=True, bf16=True),
    # more heads a kv head than a tile has
    dict(hq=17, hkv=1, hd=64, lens=[70, 0, 200]),
    dict(hq=40, hkv=1, hd=128, lens=[130], cap=50.0),
    dict(hq=16, hkv=1, hd=256, lens=[130, 2000]),
    dict(hq=33, hkv=1, hd=256, lens=[90, 1], inter=True),
    # more sequences than a wave has lanes, some of them none
    dict(hq=2, hkv=1, hd=64, lens=[(7 * i) % 150 if i % 9 else -1 for i in range(150)]),
    # windows: one row, within a page, over pages, longer than all
    dict(hq=4, hkv=2, hd=128, lens=[200, 64, 0, 63], window=1),
    dict(hq=4, hkv=2, hd=128, lens=[200, 64, 0, 90], window=2),
    dict(hq=4, hkv=2, hd=64, lens=[200, 64, 0, 1000], window=33),
    dict(hq=4, hkv=2, hd=80, lens=[200, 64, 0, 1000], window=64, cap=20.0),
    dict(hq=4, hkv=2, hd=128, lens=[200, 640, 0, 1000], window=129),
    dict(hq=4, hkv=2, hd=128, lens=[200, 64, 5], window=5000),
    # one long sequence among short ones; no rotation
    dict(hq=4, hkv=1, hd=128, lens=[5, 9000, 17, 0, 64], rope=False),
    dict(hq=4, hkv=2, hd=128, lens=[700, 650, 130], shared=2),
    # scores far apart
    dict(hq=4, hkv=2, hd=128, lens=[800, 70], std=6.0, norm=False),
]


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("kw", DECODE, ids=lambda kw: "-".join("%s" % v for v in list(kw.values())[:3]) + "-%d" % len(kw["lens"]) + "".join(
    "-%s%s" % (k, kw[k]) for k in list(kw)[4:]))
def test_decode(sa, ctx, kw, codes):
    s = Step(sa, ctx, codes=codes, **kw)
    print(kw, flush=True)
    out = torch.full((s.n, s.hq * s.hd), 777.0, device="cuda")
    s.call(out=out)
    ctx.synchronize()
    s.check(out)
    for i, l in enumerate(s.lens):
        assert l >= 0 or (out[i] == 777.0).all()  # what is no sequence stays as it was


TOP = [
    dict(hq=4, hkv=2, hd=64, lens=[0, 1, 64, 65, 300], top=4),
    dict(hq=16, hkv=8, hd=128, lens=[1000, 3000, 90, 511], top=5, first=2, recent=3),
    dict(hq=8, hkv=1, hd=256, lens=[700, 2000], top=9, first=0, inter=True, cap=30.0),
    dict(hq=15, hkv=5, hd=80, lens=[1500], top=1, first=0, norm=False),
    dict(hq=2, hkv=2, hd=72, lens=[640, 641, 639], top=8, first=1, recent=7, inter=True, bf16=True),
    dict(hq=17, hkv=1, hd=96, lens=[1300, -1, 20], top=6),
    # a table longer than what the choice keeps on the chip
    dict(hq=2, hkv=1, hd=64, lens=[900, 5], top=3, stride=5000, rope=False),
    dict(hq=2, hkv=1, hd=64, lens=[8000, 8001, 12], top=20, std=4.0),
    dict(hq=6, hkv=2, hd=128, lens=[70000, 65000], top=30, stride=2000),
    dict(hq=2, hkv=1, hd=72, lens=[5000, 300], top=30, stride=1100, rope=False),
]


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("kw", TOP, ids=lambda kw: "%d-%d-%d-top%d-%s" % (kw["hq"], kw["hkv"], kw["hd"], kw["top"], kw["lens"][0]))
def test_top(sa, ctx, kw, codes):
    s = Step(sa, ctx, codes=codes, **kw)
    print(kw, flush=True)
    out = s.call()
    ctx.synchronize()
    s.check(out, what=" top")


@pytest.mark.parametrize("stride", [None, 4200])
def test_top_ties_and_numbers_that_are_none(sa, ctx, stride):
    """pages with the same bounds: the lower ones; bounds that are no numbers count above all but the fixed pages"""
    s = Step(sa, ctx, hq=4, hkv=2, hd=128, lens=[64 * 40, 64 * 300 + 5], codes=False, top=12, first=1, recent=2, stride=stride)
    b = s.pool.views[3]
    b[:, :, 0], b[:, :, 1] = -1.0, 1.0
    b[int(s.t[1, 77]), 1, 1, 5] = math.nan
    b[int(s.t[1, 200]), 0, :, :] = 2.0
    s.before = s.pool.bits()
    s.call()
    ctx.synchronize()
    got = s.chosen.tolist()
    assert got[0][0] == got[0][1] == list(range(10)) + [38, 39]
    assert got[1][1] == list(range(9)) + [77, 299, 300]
    q = s.turned()[0]
    for h in range(2):
        assert got[1][h] == s.choose(1, h, q[1].view(2, 2, 128)[h])


# ------------------------------------------------------------------ what goes wrong

@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("top", [0, 3])
def test_numbers_out_of_range(sa, ctx, codes, top):
    """a page number or a length that is none: NaN for that sequence, an error at the next synchronize, nothing of it written"""
    for what in ("page", "past", "new page", "length"):
        s = Step(sa, ctx, hq=4, hkv=2, hd=128, lens=[500, 130, 64], codes=codes, top=top)
        if what == "page":
            s.td[1, 1] = -1
            if top:  # both of its pages are chosen
                assert s.lens[1] // P < top
        elif what == "past":
            s.td[1, 0] = s.pool.n
        elif what == "new page":
            s.lens[1] = 128
            s.ld[1] = 128
            s.td[1, 2] = 2 ** 31 - 1
        else:
            s.ld[1] = s.td.shape[1] * P
        print("out of range:", what, flush=True)
        out = s.call()
        with pytest.raises(sa.SmolAttnPageError):
            ctx.synchronize()
        ctx.synchronize()  # reported once
        assert out[1].isnan().all(), what
        keep = s.lens
        if what in ("page", "past"):
            after = s.pool.bits()  # the new row of sequence 1 has a page and is written
            s.lens = [keep[0], -1, keep[2]]
            s.check(out, stored=False, what=" beside " + what)
            assert not torch.equal(after[0], s.before[0])
        else:
            s.lens = [keep[0], -1, keep[2]]
            s.check(out, what=" beside " + what)


def test_rows_out_of_range(sa, ctx):
    g = torch.Generator().manual_seed(2)
    hkv, hd = 2, 64
    for codes in (False, True):
        t = torch.tensor([[0, 1], [2, 99], [3, 4]], dtype=torch.int32).cuda()
        k, v = normal(g, 100, hkv * hd).cuda(), normal(g, 100, hkv * hd).cuda()
        for what, starts, pos, wrote in (
                ("page", [0, 10, 90, 100], [5, 30, 0], [(0, 10, 5), (2, 34, 30), (3, 10, 0)]),
                ("end", [0, 10, 90, 101], [5, 0, 0], [(0, 10, 5)]),
                ("falls", [0, 20, 10, 15], [0, 0, 60], [(0, 20, 0), (3, 4, 60), (4, 1, 0)]),
                ("position", [0, 10, 20, 30], [120, -1, 0], [(3, 10, 0)])):
            pool = Pool(sa, ctx, 6, hkv, hd, codes, g)
            before = pool.bits()
            print("rows out of range:", what, codes, flush=True)
            sa.pages_append(pool.pool, 1, None, t, i32(starts), i32(pos), k, v)
            with pytest.raises(sa.SmolAttnPageError):
                ctx.synchronize()
            after = pool.bits()
            touched = {w[0] for w in wrote}
            for p in range(6):
                same = torch.equal(after[0][p], before[0][p])
                assert same == (p not in touched and not (what == "end" and p == 2)), (what, p)
            a = torch.full((100, hkv * hd), 5.0, device="cuda")
            b = a.clone()
            sa.pages_read(pool.pool, 1, t, i32(starts), i32(pos), 100, k_out=a, v_out=b)
            with pytest.raises(sa.SmolAttnPageError):
                ctx.synchronize()
            if what == "page":
                assert a[10 + 34:90].isnan().all() and b[10 + 34:90].isnan().all() and a[:44].isfinite().all()
            if what == "end":
                assert (a[90:] == 5.0).all()


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_rows_that_are_not_finite(sa, ctx, codes, cap):
    """one spoiled element of a visible row makes NaN of the heads that read it and of no other; behind a length and before a
    window it does nothing"""
    for where, bad in (("k", math.inf), ("k", -math.inf), ("k", math.nan), ("v", math.inf), ("v", math.nan)):
        s = Step(sa, ctx, hq=6, hkv=3, hd=128, lens=[200, 330, 64], codes=codes, cap=cap, window=150, seed=4)
        k, v, sc, _ = s.pool.views
        page, row = int(s.t[1, 300 // P]), 300 % P     # visible, of sequence 1, kv head 2
        hidden = [(int(s.t[0, 200 // P]), 200 % P + 3), (int(s.t[1, 180 // P]), 179 % P), (int(s.t[2, 1]), 10)]
        for p, r in [(page, row)] + hidden:
            if codes:
                sc[p, 2, 0 if where == "k" else 1, r] = math.nan if bad < 0 else bad
            elif where == "k":
                k[p, 2, 3, r, 5] = bad
            else:
                a = int(order(False)[r])
                v[p, 2, a // 32, 77, a % 32] = bad
        print("spoiled", where, bad, codes, cap, flush=True)
        out = s.call().cpu().view(3, 3, 2, 128)
        ctx.synchronize()
        assert out[1, 2].isnan().all()
        for i in range(3):
            for h in range(3):
                assert (i, h) == (1, 2) or out[i, h].isfinite().all(), (i, h)
    for name in ("q", "k_new", "v_new"):
        s = Step(sa, ctx, hq=6, hkv=3, hd=128, lens=[200, 330, 64], codes=codes, cap=cap, norm=False)
        s.dev[0][name].view(3, -1, 128)[1, 1, 9] = math.inf
        print("spoiled", name, codes, cap, flush=True)
        out = s.call().cpu().view(3, 6, 128)
        ctx.synchronize()
        spoiled = {1} if name == "q" else {2, 3}
        for i in range(3):
            for h in range(6):
                assert (out[i, h].isnan().all() if i == 1 and h in spoiled else out[i, h].isfinite().all()), (name, i, h)


# ------------------------------------------------------------------ as a server runs it

@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("top", [0, 4])
def test_captured_and_replayed(sa, codes, top):
    """a captured step replays with the lengths, tables and inputs of the moment, between eager calls of the same context"""
    side = torch.cuda.Stream()
    ctx = sa.Context(0, stream=side.cuda_stream)
    a = Step(sa, ctx, hq=4, hkv=2, hd=128, lens=[300, 10, -1, 700], codes=codes, top=top)
    other = Step(sa, ctx, hq=8, hkv=2, hd=64, lens=[90, 1500], codes=codes, seed=9)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        out = torch.zeros((4, 4 * 128), device="cuda")
        a.call(out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            a.call(out=out)
        for lens in ([300, 10, -1, 700], [64, 0, 5, 699], [1, 255, 200, 3], [300, -1, -1, 64]):
            b = Step(sa, ctx, hq=4, hkv=2, hd=128, lens=[max(x, y) for x, y in zip([300, 255, 200, 700], lens)], codes=codes, top=top,
                     seed=sum(lens) + 20)
            a.td[:] = -1
            pool = a.pool
            # the pages of the new table: any of the captured pool's, each once
            needs = [l // P + 1 if l >= 0 else 0 for l in lens]
            t = table_of(torch.Generator().manual_seed(7), pool.n, needs, a.t.shape[1], bad=-1)
            a.td.copy_(t)
            a.ld.copy_(torch.tensor(lens, dtype=torch.int32))
            for name in ("q", "k_new", "v_new"):
                a.dev[0][name].copy_(b.dev[0][name])
            a.q, a.k, a.v, a.t, a.lens = b.q, b.k, b.v, t, lens
            side.synchronize()
            a.before, a.rows = pool.bits(), pool.rows()
            out.fill_(777.0)
            graph.replay()
            ctx.synchronize()
            if top:
                want = out.clone()
                chosen = a.chosen
                a.check(want, what=" replay")
                assert chosen is a.chosen
            else:
                a.check(out, what=" replay")
            for i, l in enumerate(lens):
                assert l >= 0 or (out[i] == 777.0).all()
            got = other.call()
            ctx.synchronize()
            other.check(got, stored=False)
    ctx.close()


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
def test_a_batch_of_nobody(sa, ctx, codes):
    """a captured size without a request: nothing is read or written"""
    for top in (0, 2):
        s = Step(sa, ctx, hq=4, hkv=2, hd=64, lens=[-1] * 70, codes=codes, top=top)
        out = torch.full((70, 4 * 64), 3.0, device="cuda")
        s.call(out=out)
        ctx.synchronize()
        assert (out == 3.0).all()
        for a, b in zip(s.before, s.pool.bits()):
            assert a is None or torch.equal(a, b)


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
def test_two_streams(sa, codes):
    """two contexts on two streams, neither of them the current one, calls of both under way at once; the same step again gives the
    same bits"""
    runs = []
    for i in range(2):
        side = torch.cuda.Stream()
        c = sa.Context(0, stream=side.cuda_stream)
        runs.append((side, c, Step(sa, c, hq=8, hkv=2, hd=128, lens=[4000 + 100 * i, 9, 2000], codes=codes, top=8 * i, seed=30 + i)))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, (side, c, s) in enumerate(runs):
            with torch.cuda.stream(side):
                outs[i].append(s.call())
    for i, (side, c, s) in enumerate(runs):
        c.synchronize()
        s.check(outs[i][0])
        for o in outs[i][1:]:
            assert torch.equal(o, outs[i][0])
        c.close()


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
def test_what_the_products_carry(sa, ctx, codes):
    """The error of a row of out against its own norm. Scores: Q whole or at 2^-24 of its largest element, fp32 sums: their errors are random,
    about sqrt(hd) 2^-24 of |q| |k| scale (here at most 3), so 2^-20 on a weight; weights at 2^-24; the sum over 1000 rows in fp32
    2^-20. With a root of two for numerator and denominator and twice that to spare: 2^-18. Two parts of 8 bits for Q or
    the weights would leave 2^-16 of each."""
    s = Step(sa, ctx, hq=4, hkv=2, hd=128, lens=[1000, 1001, 64], codes=codes, norm=False)
    out = s.call().cpu().double().view(3, 2, 2, 128)
    ctx.synchronize()
    q, k, v = s.turned()
    kk, vv = s.rows
    for i, l in enumerate(s.lens):
        for h in range(2):
            at = torch.arange(l)
            page = s.t[i, at // P].long()
            o, _ = attend(q[i].view(2, 2, 128)[h], torch.cat([kk[page, h, at % P], k[i, h:h + 1]]),
                          torch.cat([vv[page, h, at % P], v[i, h:h + 1]]), s.scale, 0.0, codes, 128, torch.zeros(l + 1))
            err = (out[i, h] - o).norm(dim=-1) / o.norm(dim=-1)
            print("codes %d: %.2g" % (codes, float(err.max())), flush=True)
            assert (err <= 2.0 ** -18).all()


def test_growth_under_capture_is_refused(sa):
    side = torch.cuda.Stream()
    ctx = sa.Context(0, stream=side.cuda_stream)
    s = Step(sa, ctx, hq=4, hkv=2, hd=128, lens=[30, 10], codes=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(sa.SmolAttnError, match="under stream capture"):
                s.call()
            torch.zeros(4, device="cuda").add_(1)
        out = s.call()
        ctx.synchronize()
        s.check(out)
    ctx.close()


def test_a_pool_under_capture_is_refused(sa):
    """its clearing would be part of the graph"""
    side = torch.cuda.Stream()
    ctx = sa.Context(0, stream=side.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(sa.SmolAttnError, match="under stream capture"):
                sa.KVPages(ctx, 1, 4, 2, 64)
            torch.zeros(4, device="cuda").add_(1)
    ctx.close()


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
def test_choices_not_wanted(sa, ctx, codes):
    """without an array for them the step is the same; more pages than the table can have are all of them"""
    s = Step(sa, ctx, hq=4, hkv=2, hd=64, lens=[700, 64, 0, 390], codes=codes, top=4)
    a = s.call()
    ctx.synchronize()
    s.check(a, what=" top")
    d, w = s.dev
    p = lambda x: x.data_ptr()  # noqa: E731
    for top in (4, 2 ** 24 - 1):
        out = torch.empty_like(a)
        assert sa.load().smol_attn_decode_paged_top(
            ctx.h, s.pool.pool.h, s.pool.layer, s.rope.h, s.n, p(s.td), s.td.shape[1], p(s.ld), top, 1, 1, p(d["q"]), p(d["k_new"]),
            p(d["v_new"]), 0, s.hq, s.scale, 0.0, p(w["q_norm"]), p(w["k_norm"]), EPS, None, p(out)) == 0
        ctx.synchronize()
        if top == 4:
            assert torch.equal(out, a)
    s.top = 0
    s.check(out, stored=False)


def test_pool_past_four_gigabytes(sa, ctx):
    """pages whose addresses pass 32 bits"""
    hkv, hd = 8, 256
    n = 5 * 2 ** 30 // (hkv * P * hd * 2)
    pool = sa.KVPages(ctx, 1, n, hkv, hd, sa.BF16)
    g = torch.Generator().manual_seed(1)
    t = torch.tensor([[n - 1, 0, n - 2]], dtype=torch.int32).cuda()
    k, v = normal(g, 130, hkv * hd, bf16=True), normal(g, 130, hkv * hd, bf16=True)
    starts, pos = i32([0, 130]), i32([0])
    sa.pages_append(pool, 0, None, t, starts, pos, k.cuda(), v.cuda())
    a, b = sa.pages_read(pool, 0, t, starts, pos, 130)
    assert torch.equal(a.cpu(), k) and torch.equal(b.cpu(), v)
    q, kn, vn = normal(g, 1, 8 * hd), normal(g, 1, hkv * hd), normal(g, 1, hkv * hd)
    out = sa.decode_paged(ctx, pool, 0, None, t, i32([130]), q.cuda(), kn.cuda(), vn.cuda(), 8, hd ** -0.5).cpu().double()
    ctx.synchronize()
    kk = torch.cat([k.double(), kn.double()]).view(131, hkv, hd)
    vv = torch.cat([v.double(), vn.double()]).view(131, hkv, hd)
    for h in range(hkv):
        o, tol = attend(q.double().view(8, hd)[h:h + 1], kk[:, h], vv[:, h], hd ** -0.5, 0.0, False, hd, torch.zeros(131))
        assert ((out.view(8, hd)[h] - o[0]).abs() <= tol[0]).all()
    pool.close()


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
def test_a_prompt_and_its_answer(sa, ctx, codes):
    """as a server uses them together: a prompt's rows go into pages, its chunk attends to what the cache holds, tokens follow
    one by one over all rows, then over chosen pages; another sequence continues from its prefix's pages"""
    g = torch.Generator().manual_seed(3)
    hq, hkv, hd, n = 4, 2, 128, 200
    G = hq // hkv
    pool = sa.KVPages(ctx, 1, 12, hkv, hd, sa.INT8 if codes else sa.BF16)
    rope = sa.RopeTable(ctx, hd, 1e4, 0)
    t = torch.full((2, 6), -1, dtype=torch.int32)
    t[0] = torch.tensor([7, 2, 9, 4, 11, 0])
    t[1, :4] = torch.tensor([7, 2, 5, 1])     # 128 rows in common
    td = t.cuda()
    scale = hd ** -0.5
    q, k, v = (normal(g, n, h * hd) for h in (hq, hkv, hkv))
    ang = angles(sa, hd, 1e4, False, range(n))
    k64, q64 = turned(k.view(n, hkv, hd), None, ang, False), turned(q.view(n, hq, hd), None, ang, False)
    starts, pos = i32([0, n]), i32([0])
    sa.pages_append(pool, 0, rope, td[:1], starts, pos, k.cuda(), v.cuda())
    kc, vc = sa.pages_read(pool, 0, td[:1], starts, pos, n, dtype=torch.float32)
    qr = sa.norm_rope(ctx, rope, q.cuda().clone(), None, EPS, range(n), hq, hd)
    out = sa.causal(ctx, qr, kc, vc, n, n, hq, hkv, hd, scale, 0).cpu().double().view(n, hkv, G, hd)
    ctx.synchronize()
    kk, vv = kc.cpu().double().view(n, hkv, hd), vc.cpu().double().view(n, hkv, hd)
    step = 0.5 * k64.abs().amax() / 127 if codes else 2.0 ** -8 * k64.abs().amax()
    assert (kk - k64).abs().max() <= step + 2.0 ** -12
    for i in (0, 1, 63, 64, 199):
        for h in range(hkv):
            z = torch.softmax(q64[i].view(hkv, G, hd)[h] @ kk[:i + 1, h].T * scale, -1) @ vv[:i + 1, h]
            assert ((out[i, h] - z).abs() <= 2e-3 + 1e-2 * z.abs()).all()  # the bar of the path's prefill
    rows = [[(kk[j], vv[j]) for j in range(n)], [(kk[j], vv[j]) for j in range(128)]]
    lens = [n, 128]
    for turn in range(70):
        q, k, v = (normal(g, 2, h * hd) for h in (hq, hkv, hkv))
        ang = angles(sa, hd, 1e4, False, lens)
        q64, k64 = turned(q.view(2, hq, hd), None, ang, False), turned(k.view(2, hkv, hd), None, ang, False)
        v64 = v.double().view(2, hkv, hd)
        ld = i32(lens)
        args = (ctx, pool, 0, rope, td, ld, q.cuda(), k.cuda(), v.cuda(), hq, scale)
        chosen = None
        if turn % 2:
            out, chosen = sa.decode_paged_top(*args, 3)
            chosen = chosen.cpu()
        else:
            out = sa.decode_paged(*args)
        ka, va = sa.pages_read(pool, 0, td, i32([0, 1, 2]), ld, 2, dtype=torch.float32)
        ctx.synchronize()
        out = out.cpu().double().view(2, hkv, G, hd)
        for i in range(2):
            for h in range(hkv):
                use = [j for j in range(lens[i]) if chosen is None or j // P in chosen[i, h].tolist()]
                keys = torch.stack([rows[i][j][0][h] for j in use] + [k64[i, h]])
                vals = torch.stack([rows[i][j][1][h] for j in use] + [v64[i, h]])
                o, tol = attend(q64[i].view(hkv, G, hd)[h], keys, vals, scale, 0.0, codes, hd,
                                torch.tensor([j // P for j in use] + [99]))
                assert ((out[i, h] - o).abs() <= tol).all(), (turn, i, h)
            rows[i].append((ka[i].cpu().double().view(hkv, hd), va[i].cpu().double().view(hkv, hd)))
            lens[i] += 1
    pool.close()


def test_refusals(sa, ctx):
    g = torch.Generator().manual_seed(1)
    pool = sa.KVPages(ctx, 2, 4, 2, 64, sa.INT8)
    t, ld = torch.zeros((1, 2), dtype=torch.int32).cuda(), i32([5])
    q, k = normal(g, 1, 4 * 64).cuda(), normal(g, 1, 2 * 64).cuda()
    ok = dict(pages=pool, layer=0, rope=None, table=t, lens=ld, q=q, k_new=k, v_new=k.clone(), n_heads=4, scale=0.125)

    def step(match, fn=sa.decode_paged, **kw):
        with pytest.raises(sa.SmolAttnError, match=match):
            fn(ctx, **{**ok, **kw})
    step("layer 2", layer=2)
    step("not a multiple", n_heads=3, q=normal(g, 1, 3 * 64).cuda())
    step("lens must be", lens=ld.long())
    step("table must be", table=t.long())
    step("table must be", table=t[0])
    step("table must be", fn=sa.decode_paged_top, top=2, table=t[0])
    step("must be float32 or bfloat16", q=q.double())
    step("rope table head_dim", rope=sa.RopeTable(ctx, 128, 1e4))
    step("first", fn=sa.decode_paged_top, top=2, first=2)
    other = sa.Context(0)
    step("another context", pages=sa.KVPages(other, 1, 4, 2, 64))
    step("another context", rope=sa.RopeTable(other, 64, 1e4))
    for kw in (dict(n_pages=0), dict(n_layers=0), dict(n_kv_heads=0), dict(head_dim=100), dict(page_type=0), dict(page_type=3),
               dict(n_pages=2 ** 31 - 1, n_layers=2 ** 31 - 1)):
        with pytest.raises(sa.SmolAttnError):
            sa.KVPages(ctx, **{**dict(n_layers=1, n_pages=4, n_kv_heads=2, head_dim=64, page_type=sa.BF16), **kw})
    starts, pos = i32([0, 1]), i32([0])
    with pytest.raises(sa.SmolAttnError, match="starts must be"):
        sa.pages_append(pool, 0, None, t, pos, pos, k, k.clone())
    with pytest.raises(sa.SmolAttnError, match="v_new must be"):
        sa.pages_append(pool, 0, None, t, starts, pos, k, q)
    with pytest.raises(sa.SmolAttnError, match="overlap"):
        sa.pages_read(pool, 0, t, starts, pos, 1, k_out=k, v_out=k)
    sa.pages_append(pool, 0, None, t, i32([0, 0]), pos, k[:0], k[:0])  # nothing to do
    L = sa.load()
    p = lambda x: x.data_ptr()  # noqa: E731
    assert L.smol_kv_pages_read(pool.h, 0, 1, p(t), 2, p(starts), p(pos), 1, p(k), p(q), 2) == -1
    assert L.smol_kv_pages_read(pool.h, 0, 1, p(t), 2, p(starts), p(pos), 1, None, p(q), 0) == -1
    assert L.smol_kv_pages_read(pool.h, 0, 1, p(t), 0, p(starts), p(pos), 1, p(k), p(q), 0) == -1
    assert L.smol_kv_pages_read(pool.h, 0, 0, p(t), 2, p(starts), p(pos), 1, p(k), p(q), 0) == -1
    assert L.smol_kv_pages_read(pool.h, 0, 1, p(t), 2, p(starts), p(pos), -1, p(k), p(q), 0) == -1
    assert L.smol_kv_pages_append(pool.h, 0, None, 1, p(t), 2, p(starts), p(pos), 2 ** 31 - 1, p(k), p(q), 0, None, EPS) == -4
    assert L.smol_kv_pages_read(pool.h, 0, 1, p(t) + 2, 2, p(starts), p(pos), 1, p(k), p(q), 0) == -1
    assert L.smol_kv_pages_read(pool.h, 0, 1, p(t), 2, p(starts), p(pos), 1, p(k) + 8, p(q), 0) == -1
    ctx.synchronize()
    other.close()
    pool.close()
