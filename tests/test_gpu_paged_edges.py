"""Rows of a paged cache whose sizes lie far apart, against 64-bit forms: one cached row has nearly all of the softmax weight.

Bound, derived before any run. Scores are off by at most d_j = (hd + 16) 2^-24 a_j, a_j = scale max|q| sum_d |k_jd| (Q at 2^-24 of its
row's largest element or whole, its norm, rotation and scaling, the fp32 sum of the products). To first order an output moves by
sum_j p_j d_j |v_j - out|, so the row that has all of the weight moves nothing; doubled for the second order. exp, the sums, the joins and
the parts of the weights: 2^-20 sum_j p_j |v_j|. Weights of codes are 24-bit whole numbers against the largest p s of their 64 rows, each
off by half of 2^-23 / 127 of that at most, times codes of up to 127: sum over the pages of 64 127 2^-24 max(p s). s is amax / 127, and the
row's own largest code may be as low as 64: twice.
"""
import pytest

from conftest import pkg  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_paged import P, Step, ctx, order, outward, sa  # noqa: E402,F401


def set_row(s, page, h, r, k=None, v=None):
    """k and v [hd] as row r of a page of kv head h"""
    kk, vv, sc, b = s.pool.views
    o = int(order(s.codes)[r])
    for which, x in ((0, k), (1, v)):
        if x is None:
            continue
        if s.codes:
            step = x.abs().max() / 127
            sc[page, h, which, r] = step.item()
            x = (x / step).round()
        x = x.to(torch.int8 if s.codes else torch.bfloat16)
        if which:
            if s.codes:
                vv[page, h, :, o] = x.cuda()
            else:
                vv[page, h, o // 32, :, o % 32] = x.cuda()
        else:
            e = kk.shape[-1]
            kk[page, h, :, r] = torch.nn.functional.pad(x, (0, -len(x) % e)).view(-1, e).cuda()
    rows = s.pool.rows()[0][page, h].float()
    b[page, h] = torch.stack([outward(rows.amin(0), False), outward(rows.amax(0), True)]).to(torch.bfloat16).cuda()
    s.before, s.rows = s.pool.bits(), s.pool.rows()


def with_the_weight(s, at, gap, v_of):
    """row `at` of each sequence scores about `gap` with every head; v_of(i, h): its value"""
    q = s.turned()[0]
    G = s.hq // s.hkv
    for i in range(s.n):
        for h in range(s.hkv):
            u = q[i].view(s.hkv, G, s.hd)[h]
            k = (u / u.pow(2).sum(-1, keepdim=True)).sum(0) * gap / s.scale
            set_row(s, int(s.t[i, at // P]), h, at % P, k.float(), v_of(i, h))


def check(s, out, what):
    """out against 64 bits under the bound above"""
    q, k, v = s.turned()
    G, hd = s.hq // s.hkv, s.hd
    out = out.cpu().double().view(s.n, s.hkv, G, hd)
    assert torch.isfinite(out).all(), what
    worst = 0.0
    for i, l in enumerate(s.lens):
        for h in range(s.hkv):
            x, at = q[i].view(s.hkv, G, hd)[h], torch.arange(l)
            if s.top:
                pages = s.choose(i, h, x)
                assert s.chosen[i, h].tolist() == pages + [-1] * (s.top - len(pages))
                at = at[torch.isin(at // P, torch.tensor(pages))]
            page = s.t[i, at // P].long()
            keys, vals = (torch.cat([c[page, h, at % P], new[i, h:h + 1]]) for c, new in zip(s.rows, (k, v)))
            p = torch.softmax(x @ keys.T * s.scale, -1)
            o = p @ vals
            d = (hd + 16) * 2.0 ** -24 * s.scale * x.abs().amax(-1, keepdim=True) * keys.abs().sum(-1)
            tol = torch.stack([(p[g] * d[g]) @ (vals - o[g]).abs() for g in range(G)]) * 2 + 2.0 ** -20 * (p @ vals.abs())
            if s.codes:
                ps = p * vals.abs().amax(-1) / 127
                of = torch.cat([at // P, torch.tensor([-1])])
                for u in of.unique():
                    tol = tol + 2 * 64 * 127 * 2.0 ** -24 * ps[:, of == u].amax(-1, keepdim=True)
            worst = max(worst, float(((out[i, h] - o).abs() / tol).max()))
    print("%s: %.3f of the bound" % (what, worst), flush=True)
    assert worst <= 1.0


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("small,gap", [(1e-1, 25.0), (1e-3, 12.0), (1e-3, 25.0), (1e-6, 25.0), (1e-6, 40.0)])
@pytest.mark.parametrize("hq,hkv,hd", [(4, 2, 128), (3, 3, 80), (8, 1, 256), (2, 1, 64)])
def test_a_small_value_with_the_weight(sa, ctx, hq, hkv, hd, small, gap, top, codes):
    """the row that everything attends to has values far below the other rows' of its page"""
    s = Step(sa, ctx, hq=hq, hkv=hkv, hd=hd, lens=[700, 130, 64], codes=codes, norm=False, top=top, seed=hd + 1)
    g = torch.Generator().manual_seed(3)
    with_the_weight(s, 5, gap, lambda i, h: torch.randn(hd, generator=g) * small)
    out = s.call()
    ctx.synchronize()
    check(s, out, "small %g gap %g hd %d codes %d top %d" % (small, gap, hd, codes, top))


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("what", ["spread", "zeros", "tiny"])
def test_values_of_all_sizes(sa, ctx, what, codes):
    """every seventh row with values of 1e-9 to 1e9, or zero; or all values near 1e-25"""
    s = Step(sa, ctx, hq=4, hkv=2, hd=128, lens=[500, 65, 3], codes=codes, norm=False, seed=8)
    g = torch.Generator().manual_seed(4)
    for i, l in enumerate(s.lens):
        for r in range(0, l if what == "spread" else 0, 7):
            for h in range(2):
                set_row(s, int(s.t[i, r // P]), h, r % P, v=torch.randn(128, generator=g) * 10.0 ** float(18 * torch.rand(1, generator=g) - 9))
    if what == "zeros":
        if codes:
            s.pool.views[2][:, :, 1, ::7] = 0
        else:
            s.pool.views[1][..., ::7] = 0
    if what == "tiny":
        (s.pool.views[2][:, :, 1] if codes else s.pool.views[1]).mul_(1e-25)
        s.v *= 1e-25
        s.dev[0]["v_new"].mul_(1e-25)
    s.before, s.rows = s.pool.bits(), s.pool.rows()
    out = s.call()
    ctx.synchronize()
    check(s, out, "sizes %s codes %d" % (what, codes))


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("hq,hkv,hd,lens", [(4, 2, 128, [40, 64, 130]), (4, 2, 128, [6000, 70]), (2, 2, 72, [33, 900]), (8, 1, 256, [2500, 65]),
                                            (16, 1, 256, [3000, 6]), (17, 1, 64, [1500, 9])])
def test_large_finite_values(sa, ctx, hq, hkv, hd, lens, codes):
    """values whose sum over a few dims passes the largest fp32 number, though none of them does: of a cached row, of the new one"""
    for new in (False, True):
        s = Step(sa, ctx, hq=hq, hkv=hkv, hd=hd, lens=lens, codes=codes, norm=False, seed=hd + 2, rope=False)
        g = torch.Generator().manual_seed(6)
        huge = lambda *shape: (torch.randint(0, 2, shape, generator=g) * 2 - 1) * 1.2e38  # noqa: E731
        if new:  # the new row has the weight: its key is along its heads' queries
            q = s.turned()[0].view(s.n, hkv, hq // hkv, hd)
            s.k = ((q / q.pow(2).sum(-1, keepdim=True)).sum(2) * 40 / s.scale).float().view(s.n, -1)
            s.v = huge(s.n, hkv * hd)
            s.dev[0]["k_new"].copy_(s.k)
            s.dev[0]["v_new"].copy_(s.v)
        else:
            with_the_weight(s, 5, 40.0, lambda i, h: huge(hd))
        out = s.call()
        ctx.synchronize()
        check(s, out, "large, %s, hd %d codes %d" % ("new" if new else "cached", hd, codes))


@pytest.mark.parametrize("top", [1, 3, 40])
def test_choices_of_a_length_that_is_none(sa, ctx, top):
    """no page is chosen where a length is past the table's end, and nothing is written where it is negative"""
    s = Step(sa, ctx, hq=4, hkv=2, hd=64, lens=[1500, 130, -1, 64], codes=True, top=top, first=0, seed=12)
    for none in (s.td.shape[1] * P, 2 ** 31 - 1):
        s.ld[1] = none
        chosen = torch.full((s.n, s.hkv, top), 777, dtype=torch.int32, device="cuda")
        out = torch.full((s.n, s.hq * s.hd), 777.0, device="cuda")
        s.call(out=out, chosen=chosen)
        with pytest.raises(sa.SmolAttnPageError):
            ctx.synchronize()
        assert (chosen[1] == -1).all() and out[1].isnan().all()
        assert (chosen[2] == 777).all() and (out[2] == 777.0).all()
        for i in (0, 3):
            pages = -(-s.lens[i] // P)
            assert ((chosen[i] >= 0).sum(-1) == min(top, pages)).all() and (chosen[i] < pages).all()


@pytest.mark.parametrize("hq,hkv,hd", [(2, 2, 128), (4, 2, 64), (8, 1, 256), (3, 3, 72)])
@pytest.mark.parametrize("sign", [1, -1])
def test_infinite_bounds(sa, ctx, hq, hkv, hd, sign):
    """A row with an infinite element leaves an infinite bound, which counts for the heads that pick it and not for others: a page stays
    unchosen whose infinity the heads' queries all turn away from, and is chosen (and spoils the head) where one turns towards it."""
    s = Step(sa, ctx, hq=hq, hkv=hkv, hd=hd, lens=[64 * 40, 64 * 21 + 9], codes=False, norm=False, top=6, seed=hd + 3)
    q = s.turned()[0].view(s.n, hkv, hq // hkv, hd)
    b = s.before[3].view(torch.bfloat16)
    away, towards = [], []
    for i in range(s.n):
        for h in range(hkv):
            pages = -(-s.lens[i] // P)
            bb = b[s.t[i, :pages].long(), h].double()
            score = sum(torch.maximum(bb[:, 0] * x, bb[:, 1] * x).sum(-1) for x in q[i, h])
            low = int(score[1:pages - 1].argmin()) + 1     # neither fixed nor among the best
            all_away = (sign * q[i, h] < 0).all(0).nonzero()[:, 0].tolist()
            d = all_away[0] if all_away and (i + h) % 3 else int((sign * q[i, h] > 0).any(0).nonzero()[0])
            (away if d in all_away else towards).append((i, h))
            k = s.pool.views[0]
            k[int(s.t[i, low]), h, d // 8, 11, d % 8] = sign * float("inf")
            s.pool.views[3][int(s.t[i, low]), h, 1 if sign > 0 else 0, d] = sign * float("inf")
    s.before, s.rows = s.pool.bits(), s.pool.rows()
    out = s.call().cpu().view(s.n, hkv, -1)
    ctx.synchronize()
    assert towards
    for i in range(s.n):
        for h in range(hkv):
            assert s.chosen[i, h].tolist() == s.choose(i, h, q[i, h]), (i, h)
            assert out[i, h].isfinite().all() == ((i, h) in away) and out[i, h].isnan().all() == ((i, h) in towards), (i, h)


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
def test_a_bad_page_that_is_scored_only(sa, ctx, codes):
    """a page number that is none is reported also where pages without numbers for bounds take all places before it"""
    s = Step(sa, ctx, hq=4, hkv=2, hd=128, lens=[64 * 40, 64 * 3], codes=codes, top=4, first=1, recent=1, seed=15)
    for j in (1, 2):
        s.pool.views[3][int(s.t[0, j])] = float("nan")
    s.before = s.pool.bits()
    s.call()
    ctx.synchronize()
    assert s.chosen[0].tolist() == [[0, 1, 2, 39]] * 2
    for page in (-1, s.pool.n, 2 ** 31 - 1):
        s.td[0, 17] = page
        out = s.call()
        with pytest.raises(sa.SmolAttnPageError):
            ctx.synchronize()
        assert s.chosen[0].tolist() == [[0, 1, 2, 39]] * 2 and out.isfinite().all()


def append_pages(sa, ctx, pages_of_rows, hd, codes):
    """a sequence whose pages hold the rows [64, hd] given, written by the append, and its table"""
    n = len(pages_of_rows)
    pool = sa.KVPages(ctx, 1, n + 1, 1, hd, sa.INT8 if codes else sa.BF16)
    t = torch.arange(n + 1, dtype=torch.int32).flip(0)[None].contiguous().cuda()
    rows = torch.cat(pages_of_rows).cuda()
    at = torch.tensor([0, n * P], dtype=torch.int32).cuda()
    sa.pages_append(pool, 0, None, t, at, at[:1].clone(), rows, rows.clone())
    return pool, t, at


@pytest.mark.parametrize("codes", [False, True], ids=["bf16", "int8"])
def test_what_the_choice_promises(sa, ctx, codes):
    """no row of a page left out scores above the value of a page chosen by it; a page of lower scores and wider bounds may be chosen"""
    hd = 64
    g = torch.Generator().manual_seed(17)
    narrow, wide = torch.zeros(P, hd), torch.zeros(P, hd)
    narrow[:, :2] = 1.0                    # scores 2, value 2
    wide[::2, 0], wide[::2, 1] = 10.0, -10.0
    wide[1::2, 0], wide[1::2, 1] = -10.0, 10.0  # scores 0, value 20
    pool, t, at = append_pages(sa, ctx, [narrow, wide, torch.zeros(P, hd)], hd, codes)
    q, new = torch.zeros(1, hd), torch.zeros(1, hd).cuda()
    q[0, :2] = 1.0
    _, chosen = sa.decode_paged_top(ctx, pool, 0, None, t, at[1:].clone(), q.cuda(), new, new.clone(), 1, 1.0, 2, first=0, recent=1)
    assert chosen.tolist() == [[[1, 2]]]
    pool.close()
    n, top, G = 40, 9, 3
    pages = [torch.randn(P, hd, generator=g) * float(torch.rand(1, generator=g) + 0.1) + 0.5 * torch.randn(hd, generator=g) for _ in range(n)]
    pool, t, at = append_pages(sa, ctx, pages, hd, codes)
    k, _ = sa.pages_read(pool, 0, t, at, at[:1].clone(), n * P, dtype=torch.float32)
    q = torch.randn(1, G * hd, generator=g)
    _, chosen = sa.decode_paged_top(ctx, pool, 0, None, t, at[1:].clone(), q.cuda(), new, new.clone(), G, 0.125, top, first=1, recent=2)
    ctx.synchronize()
    by_value = [j for j in chosen[0, 0].tolist() if 1 <= j < n - 2]
    assert len(by_value) == top - 3
    x = 0.125 * q.double().view(G, hd)
    b = pool.views(0)[3].cpu()[t[0, :n].cpu().long(), 0].double()
    value = sum(torch.maximum(b[:, 0] * h, b[:, 1] * h).sum(-1) for h in x)
    score = (k.cpu().double() @ x.T).sum(-1).view(n, P).amax(-1)
    left = [j for j in range(1, n - 2) if j not in by_value]
    assert (score <= value + 1e-12).all()
    assert max(float(score[j]) for j in left) <= min(float(value[j]) for j in by_value)
    pool.close()


def test_a_new_pool_is_cleared_before_it_is_filled(sa):
    """its clearing, behind other work of the context's stream, does not undo what another stream writes to the new pages"""
    side = torch.cuda.Stream()
    c = sa.Context(0, stream=side.cuda_stream)
    with torch.cuda.stream(side):
        x = torch.randn(4096, 4096, device="cuda")
        for _ in range(50):
            x = torch.nn.functional.normalize(x @ x)
    pool = sa.KVPages(c, 1, 8, 2, 64, sa.INT8)
    views = pool.views(0)
    for v in views:
        v.fill_(3)
    torch.cuda.current_stream().synchronize()
    c.synchronize()
    for v in views:
        assert (v == 3).all()
    pool.close()
    c.close()


@pytest.mark.parametrize("top", [0, 4])
def test_a_graph_outlives_growth(sa, top):
    """a captured step replays after calls with a wider page table and more sequences grew the RoPE table and the workspace"""
    side = torch.cuda.Stream()
    c = sa.Context(0, stream=side.cuda_stream)
    s = Step(sa, c, hq=4, hkv=2, hd=128, lens=[900, 700, 12], codes=True, top=top, seed=41)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        out = torch.zeros((3, 4 * 128), device="cuda")
        s.call(out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s.call(out=out)
        cap = s.rope.capacity
        big = Step(sa, c, hq=4, hkv=2, hd=128, lens=[50 * i for i in range(90)], codes=True, top=top, seed=42, stride=1500)
        big.rope = s.rope
        torch.cuda.synchronize()
        for turn in range(3):
            big.call()
            c.synchronize()
            assert s.rope.capacity > cap
            # memory that was freed would hold these by now
            junk = [torch.full((n,), float("nan"), device="cuda") for n in (1 << 17, 1 << 18, 1 << 20, 1 << 22)]
            s.pool.views[3].copy_(s.before[3].view(torch.bfloat16))
            out.fill_(777.0)
            side.synchronize()
            graph.replay()
            c.synchronize()
            s.check(out, stored=False, what=" replay %d" % turn)
            del junk
    c.close()
