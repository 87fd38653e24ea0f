"""The serving operators carry fp32 operands whole through bf16 products: three parts of 8 bits each. Dense random data
hides the loss of a part behind the bound of a long fp32 sum, so here every output is ONE product: the bounds are a few
dozen roundings and smaller than what two parts leave out.

Unit: 2^-24, half a step of fp32. A sum on the matrix cores is counted with a whole step (2 units) for each term.

Attention. Key j has one element c = +-1, at dim j, and value j is one, at dim j: out_j = p_j / L, with
s_j = scale q_j c. A score: scale log2 e and its product with q 1 unit each, three parts 6: 8 |s| in all. s - m: 2 s_max.
exp 2. Products of p's three parts with one 6, rescaling 4, the waves' join 3, the chunks' 3: the numerator is off by
10 s_max + 18. The denominator: 10 s_max + 2, a lane's sums 16, four lanes 2, rescaling 4, the waves' join 7, the chunks'
11. The division 5. Together 20 s_max + 65 units; a mass is the sum of G of them (1 / L is the division): G + 4 more.
Two parts leave up to half a step of the second, 2^-17 of the value (128 units), of p; of q 2^-17 |s|.

Adapters. t = a1 x1 + a2 x2 of positive numbers: six terms 12 units, partial sums 2, scale 1; y = b t: three terms 6:
21 units. y = w x: three terms 6, and 2 for the sum over the waves. Two parts of x or t leave up to 128.
"""
import math

import pytest

from conftest import pkg  # noqa: F401

torch = pytest.importorskip("torch")

from test_gpu_adapters import Case  # noqa: E402
from test_gpu_shared import EPS, Scored, Shared, attend, ctx, err, sa  # noqa: E402,F401

U = 2.0 ** -24


def att_bound(s_max):
    return (20 * s_max + 65) * U


def parts(x, n):
    """the first n bf16 parts of fp32 x, added up"""
    total = torch.zeros_like(x, dtype=torch.float64)
    for _ in range(n):
        p = x.to(torch.bfloat16).float()
        total += p.double()
        x = x - p
    return total


@pytest.mark.parametrize("q_parts,p_parts,s_max,holds", [(3, 3, 0.5, True), (3, 3, 8.0, True), (3, 2, 0.5, False), (2, 3, 8.0, False)])
def test_the_bound_tells_two_parts_from_three(q_parts, p_parts, s_max, holds):
    """the kernel's arithmetic on the CPU, with all of its parts and with one less"""
    torch.manual_seed(1)
    q = torch.rand(64, 128) * 0.75 + 0.25
    f = torch.tensor(s_max * math.log2(math.e), dtype=torch.float64).float()
    s2 = parts(q * f, q_parts).float()
    p = torch.exp2(s2 - s2.max(-1, keepdim=True).values)
    out = parts(p, p_parts) / p.double().sum(-1, keepdim=True)
    want = torch.softmax(q.double() * s_max, -1)
    worst = float(((out - want).abs() / want).max())
    assert (worst <= att_bound(s_max)) == holds, worst / U


@pytest.mark.parametrize("x_parts,t_parts,holds", [(3, 3, True), (2, 3, False), (3, 2, False)])
def test_the_adapters_bound_tells_two_parts_from_three(x_parts, t_parts, holds):
    torch.manual_seed(1)
    x = torch.rand(64, 2, 100) * 0.75 + 0.25
    a, b = ((torch.rand(s) * 0.75 + 0.25).to(torch.bfloat16).double() for s in ((2, 100), (100,)))
    t = (parts(x, x_parts) * a).sum(1)
    y = parts(t.float(), t_parts) * b
    want = (x.double() * a).sum(1) * b
    assert (float(((y - want).abs() / want).max()) <= 21 * U) == holds


def one_products(s, g, n_keys, kk, vv, first):
    """rows [first, first + n_keys) of a one-element key and value each: signs per row"""
    sign = torch.where(torch.rand(n_keys, generator=g) < 0.5, -1.0, 1.0)
    j = torch.arange(first, first + n_keys)
    kk[:n_keys], vv[:n_keys] = 0.0, 0.0
    kk[torch.arange(n_keys), j] = sign.to(kk.dtype)
    vv[torch.arange(n_keys), j] = 1.0


def spread_q(s, g):
    s.q[:] = (torch.rand(s.q.shape, generator=g) * 0.75 + 0.25) * torch.where(torch.rand(s.q.shape, generator=g) < 0.5, -1.0, 1.0)


def ratio(got, want, bound):
    """the worst error in bounds; outputs of keys that a sequence has not are zeros"""
    assert (got[want == 0] == 0).all()
    on = want > 0
    return float(((got[on] - want[on]).abs() / (bound * want[on])).max())


# narrow items, wide ones, every head_dim
@pytest.mark.gpu
@pytest.mark.parametrize("s_max", [0.5, 8.0], ids=["weights", "scores"])
@pytest.mark.parametrize("hq,hkv,hd,n", [(4, 2, 64, 6), (4, 1, 64, 24), (3, 1, 72, 8), (6, 2, 80, 9), (8, 2, 96, 12), (4, 2, 128, 6),
                                         (8, 2, 128, 24), (17, 1, 128, 2), (4, 1, 256, 7)])
def test_shared_parts(sa, ctx, hq, hkv, hd, n, s_max):
    prefix = hd // 2 + 3
    lens = [(hd - prefix - 1, 0, 7, hd - prefix - 2)[i % 4] for i in range(n)]
    s = Shared(sa, ctx, hq, hkv, hd, lens, prefix, norm=False, rope=False)
    s.scale = s_max
    g = torch.Generator()
    g.manual_seed(hd)
    spread_q(s, g)
    new_k, new_v = s.k.view(n, hkv, hd), s.v.view(n, hkv, hd)
    for h in range(hkv):
        one_products(s, g, prefix, s.pre.k[s.p_slot, h], s.pre.v[s.p_slot, h], 0)
        for i, l in enumerate(lens):
            one_products(s, g, l, s.own.k[s.slots[i], h], s.own.v[s.slots[i], h], prefix)
            one_products(s, g, 1, new_k[i, h:h + 1], new_v[i, h:h + 1], hd - 1)
    s.pre.push()
    s.own.push()
    out = s.call().cpu().double().view(n, hkv, hq // hkv, hd)
    q, k, v = s.rows64()
    worst = 0.0
    for i, l in enumerate(lens):
        for h in range(hkv):
            kk = torch.cat([s.pre.k[s.p_slot, h, :prefix].double(), s.own.k[s.slots[i], h, :l].double(), k[i, h:h + 1]])
            vv = torch.cat([s.pre.v[s.p_slot, h, :prefix].double(), s.own.v[s.slots[i], h, :l].double(), v[i, h:h + 1]])
            want = attend(q[i].view(hkv, -1, hd)[h], kk, vv, s_max, 0.0)[0]
            worst = max(worst, ratio(out[i, h], want, att_bound(s_max)))
    print("one product an output, head_dim %d, %d rows, scores to %g: %.3f of the bound" % (hd, n * hq // hkv, s_max, worst), flush=True)
    assert worst <= 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("s_max", [0.5, 8.0], ids=["weights", "scores"])
@pytest.mark.parametrize("hq,hkv,hd", [(4, 2, 64), (2, 1, 72), (6, 2, 128), (4, 1, 256)])
def test_scored_parts(sa, ctx, hq, hkv, hd, s_max):
    rows = [hd - 1, 0, hd // 2]
    s = Scored(sa, ctx, hq, hkv, hd, rows, norm=False, decay=0.0)
    s.rope, s.scale = None, s_max
    g = torch.Generator()
    g.manual_seed(hd)
    spread_q(s, g)
    n, new_k, new_v = s.n, s.k.view(s.n, hkv, hd), s.v.view(s.n, hkv, hd)
    for h in range(hkv):
        for i, l in enumerate(rows):
            one_products(s, g, l, s.own.k[s.slots[i], h], s.own.v[s.slots[i], h], 0)
            one_products(s, g, 1, new_k[i, h:h + 1], new_v[i, h:h + 1], hd - 1)
    s.own.push()
    m, p = s.arrays()
    out = s.call(m, p).cpu().double().view(n, hkv, hq // hkv, hd)
    m = m.cpu().double()
    worst = 0.0
    for i, l in enumerate(rows):
        for h in range(hkv):
            kk = torch.cat([s.own.k[s.slots[i], h, :l].double(), new_k[i, h:h + 1].double()])
            vv = torch.cat([s.own.v[s.slots[i], h, :l].double(), new_v[i, h:h + 1].double()])
            want, w = attend(s.q.view(n, hkv, -1, hd)[i, h].double(), kk, vv, s_max, 0.0)[:2]
            worst = max(worst, ratio(out[i, h], want, att_bound(s_max)),
                        ratio(m[s.slots[i], h, :l + 1], w.sum(0), att_bound(s_max) + (hq // hkv + 4) * U))
    print("scored, one product an output, head_dim %d, scores to %g: %.3f of the bound" % (hd, s_max, worst), flush=True)
    assert worst <= 1.0


@pytest.mark.gpu
def test_shared_and_decode(sa, ctx):
    """the shared step and the decode step of sequences that hold the prefix themselves, each within its own bound: the
    decode step carries Q and the probabilities in two bf16 parts, 2^-16 of a score and of a weight"""
    s = Shared(sa, ctx, 8, 4, 128, [40, 0, 5], 333)
    out = s.call()
    kv = sa.KVCache(ctx, 1, 3, 4, 128, 512)
    for i, (sl, l) in enumerate(zip(s.slots, s.lens)):
        rk = torch.cat([s.pre.k[s.p_slot, :, :333], s.own.k[sl, :, :l]], 1)
        rv = torch.cat([s.pre.v[s.p_slot, :, :333], s.own.v[sl, :, :l]], 1)
        flat = lambda t: t.transpose(0, 1).reshape(333 + l, -1).contiguous().cuda()  # noqa: E731
        kv.write(0, i, 0, flat(rk), flat(rv))
    (q, k, v), (qw, kw) = s.dev
    two = sa.decode(ctx, kv, 0, s.rope, [0, 1, 2], [333 + l for l in s.lens], q, k, v, 8, s.scale, q_norm=qw, k_norm=kw, eps=EPS)
    q, k, v = s.rows64()
    for i, (sl, l) in enumerate(zip(s.slots, s.lens)):
        for h in range(4):
            kk = torch.cat([s.pre.k[s.p_slot, h, :333].double(), s.own.k[sl, h, :l].double(), k[i, h:h + 1]])
            vv = torch.cat([s.pre.v[s.p_slot, h, :333].double(), s.own.v[sl, h, :l].double(), v[i, h:h + 1]])
            o, _, w, a = attend(q[i].view(4, 2, 128)[h], kk, vv, s.scale, 0.0)
            e3 = err(128, a) - 2.0 ** -16 + 2.0 ** -23  # three parts of p
            e2 = err(128, a) + 2 * 2.0 ** -16 * a
            for got, e in ((out, e3), (two, e2)):
                got = got[i].cpu().double().view(4, 2, 128)[h]
                assert ((got - o).abs() <= 2 * e * w + 2.0 ** -22 * o.abs()).all(), (i, h)
    kv.close()


# one launch, two with 16, 32 and 64 rows, the library's product beside; whole and padded ranks and sizes
SIZES = [(3, 512, 70, [8, 3]), (9, 96, 70, [100, 20]), (14, 1032, 33, [16]), (20, 333, 65, [16, 40]), (50, 520, 130, [8, 17]),
         (130, 512, 96, [32, 5]), (130, 333, 70, [16, 100])]


def adapters_case(n, k, out, ranks, bf16, low):
    t = Case(n, k, out, ranks, bf16=bf16, bias=False, bare=0.0)
    g = torch.Generator()
    g.manual_seed(k)

    def number(*shape):
        return torch.rand(shape, generator=g) * 0.75 + 0.25
    t.x.copy_(number(n, k))
    t.w.zero_()
    if not low:
        t.w[torch.arange(out), torch.randint(0, k, (out,), generator=g)] = number(out).to(torch.bfloat16)
    for i, (a, b, _) in enumerate(t.ab):
        a.zero_()
        b.zero_()
        r = a.shape[0]
        if low:
            j = torch.randint(0, k // 2, (r,), generator=g)
            a[torch.arange(r), j] = number(r).to(torch.bfloat16)
            a[torch.arange(r), j + k // 2] = (number(r) * 2.0 ** -6).to(torch.bfloat16)
        b[torch.arange(out), torch.randint(0, r, (out,), generator=g)] = number(out).to(torch.bfloat16)
        t.ab[i] = (a, b, 0.5 + 0.25 * i)
    return t


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["x_f32", "x_bf16"])
@pytest.mark.parametrize("low", [True, False], ids=["low_rank", "shared"])
@pytest.mark.parametrize("n,k,out,ranks", SIZES)
def test_adapters_parts(sa, ctx, n, k, out, ranks, bf16, low):
    t = adapters_case(n, k, out, ranks, bf16, low)
    y = t.call(sa, ctx).cpu().double()
    x = t.x.double()
    if low:
        want = torch.stack([torch.tensor(t.ab[i][2]).double() * (t.ab[i][1].double() @ (t.ab[i][0].double() @ x[s]))
                            for s, i in enumerate(t.ids)])
        bound = 21 * U
    else:
        want = x @ t.w.double().T
        # more than 64 rows are the library's product, which carries an fp32 x to 2^-16
        bound = 8 * U if n <= 64 or bf16 else 8 * U + 2.0 ** -16
    worst = ratio(y, want, bound)
    print("adapters %s: %.3f of the bound" % ((n, k, out, ranks, bf16, low), worst), flush=True)
    assert worst <= 1.0
