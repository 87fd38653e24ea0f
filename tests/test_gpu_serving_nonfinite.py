"""One value that is no finite number in a visible row of the serving decode steps: the heads that read the row give NaN,
all of them, whatever the signs, the softcap and the windows; everything else keeps its bits. (A score that an infinite
key turns to -inf would drop out of the softmax, one that a softcap clips would weigh like any other.)"""
import pytest

from conftest import pkg  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_shared import Scored, Shared, ctx, sa  # noqa: E402,F401

INF, NAN = float("inf"), float("nan")

# narrow items, wide ones, head sizes with padded tiles and the largest, several blocks of a kv head's heads
SHAPES = [
    dict(hq=16, hkv=2, hd=128, lens=[40, 0, 65], prefix=100),
    dict(hq=28, hkv=2, hd=64, lens=[3, 70, 0, 33], prefix=77),
    dict(hq=24, hkv=2, hd=128, lens=[3, 70, 0, 33], prefix=300),
    dict(hq=12, hkv=2, hd=72, lens=[40, 7], prefix=50, inter=True),
    dict(hq=16, hkv=2, hd=256, lens=[40, 7], prefix=50),
    dict(hq=34, hkv=2, hd=64, lens=[40, 7], prefix=50),
]
shapes = pytest.mark.parametrize("c", SHAPES, ids=lambda c: "%d-%d-%d" % (c["hq"], c["hkv"], c["hd"]))


def heads(s, out):
    return out.view(s.n, s.hkv, s.hq // s.hkv, s.hd)


def only(s, out, clean, hit):
    """NaN in every output of the (sequence, kv head) pairs of hit, the clean call's bits in all others"""
    out, clean = heads(s, out), heads(s, clean)
    for i in range(s.n):
        for g in range(s.hkv):
            if (i, g) in hit:
                assert torch.isnan(out[i, g]).all(), (i, g, torch.isnan(out[i, g]).sum().item())
            else:
                assert torch.equal(out[i, g], clean[i, g]), (i, g)


@pytest.mark.parametrize("cap", [0.0, 30.0], ids=["", "cap"])
@shapes
def test_one_key_element(sa, ctx, c, cap):
    s = Shared(sa, ctx, cap=cap, **c)
    clean = s.call().clone()
    long = max(range(s.n), key=lambda i: s.lens[i])
    for bad, d in ((INF, 5), (-INF, s.hd - 1), (NAN, 0)):
        for row in (0, 33, s.prefix - 1):
            keep = s.pre.k[s.p_slot, 1, row, d].clone()
            s.pre.k[s.p_slot, 1, row, d] = bad
            s.pre.push()
            only(s, s.call(), clean, {(i, 1) for i in range(s.n)})
            s.pre.k[s.p_slot, 1, row, d] = keep
        s.pre.push()
        for row in (0, s.lens[long] - 1):
            at = s.own.k[s.slots[long], 0, row]
            keep = at[d].clone()
            at[d] = bad
            s.own.push()
            only(s, s.call(), clean, {(long, 0)})
            at[d] = keep
        s.own.push()
    assert torch.equal(s.call(), clean)


@shapes
def test_one_value_element(sa, ctx, c):
    s = Shared(sa, ctx, **c)
    clean = s.call().clone()
    long = max(range(s.n), key=lambda i: s.lens[i])
    for bad, d in ((INF, 5), (-INF, s.hd - 1), (NAN, 0)):
        for row in (0, 33):
            keep = s.pre.v[s.p_slot, 1, row, d].clone()
            s.pre.v[s.p_slot, 1, row, d] = bad
            s.pre.push()
            only(s, s.call(), clean, {(i, 1) for i in range(s.n)})
            s.pre.v[s.p_slot, 1, row, d] = keep
        s.pre.push()
        at = s.own.v[s.slots[long], 0, s.lens[long] - 1]
        keep = at[d].clone()
        at[d] = bad
        s.own.push()
        only(s, s.call(), clean, {(long, 0)})
        at[d] = keep
        s.own.push()
    assert torch.equal(s.call(), clean)


@pytest.mark.parametrize("where", ["k", "v"])
@shapes
def test_one_element_of_the_new_token(sa, ctx, c, where):
    s = Shared(sa, ctx, norm=False, cap=0.0 if where == "v" else 30.0, **c)
    clean = s.call().clone()
    new = s.dev[0][1 if where == "k" else 2].view(s.n, s.hkv, s.hd)
    for bad, d in ((INF, 5), (-INF, s.hd - 1), (NAN, 0)):
        keep = new[1, 1, d].clone()
        new[1, 1, d] = bad
        only(s, s.call(), clean, {(1, 1)})
        new[1, 1, d] = keep
    assert torch.equal(s.call(), clean)


@pytest.mark.parametrize("cap", [0.0, 30.0], ids=["", "cap"])
@pytest.mark.parametrize("c", [(8, 2, 64), (56, 2, 64), (24, 2, 96), (56, 2, 128)], ids=lambda c: "%d-%d-%d" % c)
@pytest.mark.parametrize("which", ["k", "v"])
def test_windows_that_differ(sa, ctx, which, c, cap):
    """rows seen: from 101, 131 and 161 on (slabs start at 96, 128, 160)"""
    s = Shared(sa, ctx, *c, [0, 30, 60], 200, window=100, cap=cap)
    clean = s.call().clone()
    side = getattr(s.pre, which)
    for bad, d in ((INF, 5), (-INF, s.hd - 1), (NAN, 0)):
        for row, who in ((100, []), (101, [0]), (130, [0]), (131, [0, 1]), (140, [0, 1]), (161, [0, 1, 2]), (199, [0, 1, 2])):
            keep = side[s.p_slot, 0, row, d].clone()
            side[s.p_slot, 0, row, d] = bad
            s.pre.push()
            only(s, s.call(), clean, {(i, 0) for i in who})
            side[s.p_slot, 0, row, d] = keep
    s.pre.push()
    assert torch.equal(s.call(), clean)


@pytest.mark.parametrize("cap", [0.0, 30.0], ids=["", "cap"])
@pytest.mark.parametrize("hq,hkv,hd", [(16, 2, 128), (12, 2, 72), (40, 2, 64), (16, 2, 256)])
def test_scored(sa, ctx, hq, hkv, hd, cap):
    """a key spoils the outputs and the weights of the kv head that reads it, a value its outputs alone"""
    s = Scored(sa, ctx, hq, hkv, hd, [70, 33, 1100], cap=cap)
    m0, p0 = s.arrays()
    clean = s.call(m0, p0).clone()
    for bad, d in ((INF, 5), (-INF, s.hd - 1), (NAN, 0)):
        for which in ("k", "v"):
            side = getattr(s.own, which)
            for i, g, row in ((0, 1, 69), (2, 0, 40), (2, 0, 1099)):
                at = side[s.slots[i], g, row]
                keep = at[d].clone()
                at[d] = bad
                s.own.push()
                m, p = s.arrays()
                only(s, s.call(m, p), clean, {(i, g)})
                n = s.rows[i] + 1
                if which == "k":
                    assert torch.isnan(m[s.slots[i], g, :n]).all()
                    m[s.slots[i], g, :n] = m0[s.slots[i], g, :n]
                assert torch.equal(m.view(torch.int32), m0.view(torch.int32)) and torch.equal(p, p0)
                at[d] = keep


def test_scores_past_the_range_drop_out(sa, ctx):
    """finite keys whose scores pass fp32's range downwards have no weight, as by the formula: not every infinite score
    is a spoiled row (a product of 6e38 does, while those of the second bf16 part, 2^-8 of it, and their sum do not)"""
    s = Shared(sa, ctx, 4, 2, 128, [40, 0], 64, norm=False, rope=False)
    s.q[:] = s.q.abs() + 1e20
    s.k[:] = 1e-20 * s.k
    s.pre.k[:] = -s.pre.k.abs() * 1e-20
    s.own.k[:] = -s.own.k.abs() * 1e-20
    s.pre.push()
    s.own.push()
    assert torch.isfinite(s.call()).all()
    s.pre.k[s.p_slot, :, 7] = -5e19
    s.pre.push()
    out = s.call()
    assert torch.isfinite(out).all()
    q, k, v = s.rows64()
    # the row that dropped out aside, the formula's result on what is left
    for i in range(s.n):
        for h in range(2):
            keep = [r for r in range(64) if r != 7]
            kk = torch.cat([s.pre.k[s.p_slot, h, keep].double(), s.own.k[s.slots[i], h, :s.lens[i]].double(), k[i, h:h + 1]])
            vv = torch.cat([s.pre.v[s.p_slot, h, keep].double(), s.own.v[s.slots[i], h, :s.lens[i]].double(), v[i, h:h + 1]])
            z = q[i].view(2, 2, 128)[h] @ kk.T * s.scale
            w = torch.softmax(z, -1)
            a = float((q[i].view(2, 2, 128)[h].abs() @ kk.abs().T * s.scale).max())
            # a score is off by at most (hd + 8) 2^-24 a, a weight by twice that, three 2^-21 for the rest
            e = 2 * (128 + 8) * 2.0 ** -24 * a + 3 * 2.0 ** -21
            assert ((out[i].cpu().double().view(2, 2, 128)[h] - w @ vv).abs() <= 2 * e * (w @ vv.abs())).all()
