"""Learned type vectors on the GPU against their definitions in 64 bits: lookup, layer norm, dropout and their gradients."""
import gc

import pytest
import torch

import libmolgrid_b200 as lmg
from libmolgrid_b200 import _cabi, api
from tests import vectors_plain as plain

pytestmark = pytest.mark.gpu

F, B, H = torch.float32, torch.bfloat16, torch.float16
RNG = (0x9e3779b97f4a7c15, 0x123456789abc)
GUARD = 17.0


def gen(seed=1):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def guarded(shape, dtype, pad=0, offset=0):
    """(array of rows ``pad`` elements further apart than they are long, ``offset`` elements into a buffer; a check that
    nothing else of the buffer changed)."""
    rows, W = 1, shape[-1]
    for n in shape[:-1]:
        rows *= n
    ld = W + pad
    buf = torch.full((offset + rows * ld + 64,), GUARD, dtype=dtype, device="cuda")
    strides, s = [1], ld
    for n in reversed(shape[:-1]):
        strides.insert(0, s)
        s *= n
    view = buf.as_strided(shape, strides, offset)

    def check():
        mask = torch.ones_like(buf, dtype=torch.bool)
        mask.as_strided(shape, strides, offset).fill_(False)
        assert bool((buf[mask] == GUARD).all()), "written beside the rows"
    return view, check


def strided(t, pad, offset=0):
    v, _ = guarded(t.shape, t.dtype, pad, offset)
    v.copy_(t)
    return v


def make_types(g, lead, V, kind, hot=False):
    t = torch.randint(0, max(V, 1), lead, generator=g, device="cuda")
    if hot:
        t = torch.where(torch.rand(lead, generator=g, device="cuda") < 0.7, torch.full_like(t, V // 2), t)
    t[torch.rand(lead, generator=g, device="cuda") < 0.1] = -1
    return t.to(kind)


def counts(g, lead):
    n = torch.randint(0, lead[1] + 1, (lead[0],), generator=g, device="cuda", dtype=torch.int32)
    n[0] = 0
    if lead[0] > 1:
        n[1] = lead[1]
    return n


LOOKUPS = [
    # lead, ntypes, width, table, vectors, index, p, pad, offset
    ((1,), 1, 1, F, F, F, 0.0, 0, 0),
    ((40,), 14, 32, F, F, F, 0.0, 0, 0),
    ((40,), 14, 32, F, F, F, 0.25, 0, 0),
    ((3, 17), 28, 28, F, F, F, 0.3, 0, 0),
    ((5, 301), 28, 45, F, H, torch.int32, 0.25, 0, 0),
    ((5, 301), 28, 45, H, H, torch.int32, 0.0, 0, 0),
    ((1000,), 3000, 33, B, B, torch.int64, 0.1, 0, 0),
    ((1000,), 3000, 3, F, B, torch.int64, 0.5, 0, 0),
    ((2, 777), 257, 100, B, B, torch.int64, 0.9, 4, 0),
    ((2, 777), 257, 100, F, F, F, 0.1, 12, 4),
    ((2, 777), 5, 7, F, F, F, 0.1, 1, 1),
    ((333,), 70001, 1, F, F, F, 0.5, 0, 1),
    ((70,), 70001, 1024, B, B, torch.int64, 0.0, 0, 0),
    ((9000,), 2, 8, F, F, torch.int32, 0.0, 0, 0),
    ((9000,), 300, 257, H, H, torch.int32, 0.2, 0, 3),
    ((6,), 11, 8200, F, H, F, 0.2, 0, 0),
    ((40000,), 28, 24, F, F, F, 0.1, 0, 0),
    ((20000,), 5000, 64, F, F, torch.int64, 0.0, 0, 0),
    ((20000,), 5000, 40, B, F, torch.int64, 0.0, 0, 0),
    ((20000,), 20000, 13, H, H, torch.int64, 0.3, 0, 0),
    ((30000,), 70001, 16, F, F, torch.int64, 0.3, 0, 0),
    ((128, 500), 90, 31, F, F, F, 0.0, 0, 0),
    # sorted in several launches
    ((40000,), 5000, 24, F, F, torch.int64, 0.2, 0, 0), ((33000,), 70001, 9, H, H, torch.int64, 0.1, 0, 0),
    ((10, 4500), 1500, 12, F, B, F, 0.0, 4, 0), ((32769,), 130, 40, F, F, torch.int32, 0.3, 0, 1),
    # few types of wide rows, which are sorted too; one slot more than a network sorts, and as many as it does
    ((3000,), 30, 300, F, F, F, 0.0, 0, 0), ((700,), 20, 1000, B, B, F, 0.3, 0, 0), ((1025,), 4000, 20, F, F, torch.int32, 0.0, 0, 0),
    ((1024,), 4000, 21, F, F, torch.int32, 0.4, 0, 0), ((1024,), 2097151, 4, F, F, torch.int32, 0.0, 0, 0),
    ((900,), 2097152, 4, F, F, torch.int32, 0.0, 0, 0), ((32768,), 113, 16, F, F, torch.int32, 0.0, 0, 0),
    # types shared out among clusters: 64 of a cluster, twice as many clusters as fit at once, and one type too many; widths and lengths at the ends
    ((5000,), 960, 8, F, F, torch.int32, 0.0, 0, 0), ((4097,), 961, 17, F, F, F, 0.2, 0, 1), ((5000,), 1920, 9, H, H, torch.int64, 0.0, 0, 0),
    ((5000,), 1921, 9, H, H, torch.int64, 0.0, 0, 0), ((1100,), 113, 1, H, H, F, 0.5, 0, 0), ((20000,), 960, 256, B, B, F, 0.2, 0, 0),
    ((1500,), 121, 256, F, B, F, 0.0, 8, 0), ((100000,), 200, 83, F, F, torch.int32, 0.0, 0, 0), ((7, 25001), 350, 40, F, H, F, 0.1, 0, 0),
    ((300000,), 350, 20, F, F, F, 0.0, 0, 0),
]
IDS = ["%s-%dx%d-%s" % ("x".join(map(str, c[0])), c[1], c[2], str(c[4])[6:]) for c in LOOKUPS]


@pytest.mark.parametrize("case", LOOKUPS, ids=IDS)
def test_lookup(case):
    lead, V, W, tt, vt, kind, p, pad, offset = case
    if tt is not F and vt is F:
        pytest.skip("a table of 16 bits has vectors of 16 bits")
    g = gen(3)
    types, table = make_types(g, lead, V, kind), strided(normal(g, V, W, dtype=tt), pad)
    na = counts(g, lead) if len(lead) == 2 else None
    out, check = guarded(lead + (W,), vt, pad, offset)
    scale = 1.5 if tt is vt and vt is not F else 0.7
    lmg.embed_types(types, table, out, scale, na, p, RNG)
    want, tol = plain.embed(types, table, scale, na, p, RNG)
    plain.assert_near(out, want, tol)
    check()
    first = out.clone()
    lmg.embed_types(types, table, out, scale, na, p, RNG)
    assert torch.equal(first, out)


@pytest.mark.parametrize("hot", [False, True], ids=["even", "hot"])
@pytest.mark.parametrize("case", LOOKUPS, ids=IDS)
def test_lookup_gradient(case, hot):
    lead, V, W, tt, vt, kind, p, pad, offset = case
    g = gen(4)
    types = make_types(g, lead, V, kind, hot)
    na = counts(g, lead) if len(lead) == 2 else None
    diff = strided(normal(g, *lead, W, dtype=tt if vt is F else vt), pad, offset)
    if tt is not F and vt is F:
        tt = F                                  # 16-bit gradients into a float32 table
    grad, check = guarded((V, W), tt, pad, offset)
    empty = plain.valid_types(types, V, na) < 0
    diff[empty] = float("nan")                  # what lies in empty slots is not read
    lmg.embed_types_backward(types, diff, grad, 0.7, na, p, RNG)
    want, tol = plain.embed_backward(types, diff, V, 0.7, na, p, RNG)
    plain.assert_near(grad, want, tol)
    check()
    first = grad.clone()
    grad.fill_(5.0)
    lmg.embed_types_backward(types, diff, grad, 0.7, na, p, RNG)
    assert torch.equal(first, grad)


@pytest.mark.parametrize("kind", [F, torch.int32, torch.int64])
def test_types_that_leave_a_slot_empty(kind):
    V, W = 4, 5
    t = [0, 3, -1, 4, -7, 2 ** 31 - 1, -(2 ** 31), 1]
    if kind is F:
        t += [float("nan"), float("inf"), -float("inf"), 2.4, 2.5, -0.4, -0.5, 3.5, 1e30]
    elif kind is torch.int64:
        t += [2 ** 40, -2 ** 40, 2 ** 32, 2 ** 32 + 1, -2 ** 32]
    types = torch.tensor(t, device="cuda", dtype=kind)
    table = normal(gen(), V, W)
    out = torch.full((len(t), W), GUARD, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lmg.embed_types(types, table, out, status=status)
    valid = plain.valid_types(types, V, None)
    assert torch.equal(out, torch.cat([table, torch.zeros(1, W, device="cuda")])[valid])
    assert int(status) == 1
    status.zero_()
    grad = torch.full((V, W), GUARD, device="cuda")
    lmg.embed_types_backward(types, torch.ones_like(out), grad, status=status)
    assert grad[:, 0].tolist() == [float((valid == v).sum()) for v in range(V)] and int(status) == 1
    status.zero_()
    lmg.embed_types(types.clamp(-1, 3) if kind is not F else types[:3], table, out if kind is not F else out[:3], status=status)
    assert int(status) == 0
    # what lies behind the atoms is no type, whatever it is
    padded = torch.tensor([[1, 2 ** 30], [2 ** 30, 2 ** 30]], device="cuda").to(kind)
    lmg.embed_types(padded, table, torch.empty(2, 2, W, device="cuda"), n_atoms=torch.tensor([1, 0], device="cuda", dtype=torch.int32),
                    status=status)
    assert int(status) == 0


def test_infinities_and_nan_stay_in_their_rows():
    table = torch.tensor([[1.0, 2.0], [float("nan"), 1.0], [float("inf"), -float("inf")]], device="cuda")
    types = torch.tensor([0, 1, 2, 0, -1], device="cuda")
    out = torch.empty(5, 2, device="cuda")
    lmg.embed_types(types, table, out)
    assert torch.equal(out[[0, 3, 4]], torch.tensor([[1.0, 2], [1, 2], [0, 0]], device="cuda"))
    assert out[1, 0].isnan() and out[2].isinf().all()
    diff = torch.zeros(5, 2, device="cuda")
    diff[1, 0], diff[2, 1] = float("nan"), float("inf")
    grad = torch.empty(3, 2, device="cuda")
    lmg.embed_types_backward(types, diff, grad)
    assert grad[1, 0].isnan() and grad[2, 1].isinf() and float(grad[0].abs().sum() + grad[1, 1] + grad[2, 0]) == 0
    x = torch.full((64, 8), float("inf"), device="cuda")
    lmg.dropout(x, x, 0.5, RNG)
    kept = plain.factors(64, 8, 0.5, RNG) != 0
    assert torch.equal(x.isinf(), kept) and bool((x[~kept] == 0).all())


NORMS = [
    # lead, width, vectors, parameters, pad, offset
    ((1,), 1, F, F, 0, 0), ((5,), 2, F, F, 0, 0), ((40,), 3, H, H, 0, 0), ((40,), 32, F, F, 0, 0), ((3, 17), 28, F, F, 0, 0),
    ((7, 133), 28, B, F, 0, 0), ((7, 133), 45, H, H, 0, 0), ((7, 133), 64, H, F, 8, 0), ((7, 133), 64, B, B, 1, 1), ((300,), 100, F, F, 0, 1),
    ((300,), 128, F, F, 4, 4), ((2, 60), 333, F, F, 0, 0), ((130,), 512, B, F, 0, 0), ((2, 60), 1001, H, H, 0, 0), ((130,), 1024, F, F, 0, 0),
    ((2, 33), 2050, B, F, 0, 0), ((33,), 4096, B, F, 0, 0), ((9,), 8192, F, F, 0, 0), ((9,), 8200, H, H, 0, 0), ((5,), 16391, F, F, 0, 0),
    ((3,), 40000, B, B, 0, 0), ((20000,), 8, F, F, 0, 0), ((3000,), 257, B, F, 0, 0), ((50000,), 28, F, F, 0, 0), ((4000,), 1032, H, F, 0, 0),
    ((700,), 505, H, H, 0, 0), ((300,), 511, F, F, 1, 1), ((2100,), 17, B, B, 0, 0), ((640,), 64, F, F, 0, 0), ((640,), 65, F, F, 0, 0),
    ((1300,), 2048, B, B, 0, 0), ((900,), 5984, B, F, 0, 0), ((170,), 8191, F, F, 0, 0), ((170,), 8185, H, H, 0, 1), ((2000,), 700, H, F, 0, 0),
]


@pytest.mark.parametrize("affine", [True, False], ids=["affine", "plain"])
@pytest.mark.parametrize("case", NORMS, ids=["%s-%d-%s-%s" % ("x".join(map(str, c[0])), c[1], str(c[2])[6:], str(c[3])[6:]) for c in NORMS])
def test_layer_norm(case, affine):
    lead, W, vt, pt, pad, offset = case
    g = gen(6)
    na = counts(g, lead) if len(lead) == 2 else None
    x = normal(g, *lead, W) * (0.5 + torch.rand(lead + (1,), generator=g, device="cuda")) + normal(g, *lead, 1)
    x = strided(x.to(vt), pad, offset)
    diff = strided(normal(g, *lead, W, dtype=vt), pad, offset)
    w = (1 + 0.3 * normal(g, W)).to(pt) if affine else None
    b = normal(g, W).to(pt) if affine else None
    if na is not None:
        x[~plain.filled(lead, na)] = float("nan")
        diff[~plain.filled(lead, na)] = float("nan")
    out, check = guarded(lead + (W,), vt, pad, offset)
    stats, check_stats = guarded(lead + (2,), F)
    lmg.layer_norm(x, w, b, out, stats, 1e-5, na)
    N = plain.Norm(x, w, b, 1e-5, na)
    plain.assert_near(out, *N.forward())
    check(), check_stats()
    on = N.on[..., 0]
    plain.assert_near(stats[on][:, :1], N.mean[on], N.dmean[on])
    assert bool(((stats[on][:, 1:].double() / N.q[on] - 1).abs() <= N.dq[on] + 2 * plain.U).all())
    bare, _ = guarded(lead + (W,), vt, pad, offset)       # last bits go by the arrays' alignment: the same call again
    lmg.layer_norm(x, w, b, bare, None, 1e-5, na)
    assert torch.equal(bare, out)
    dense = torch.empty(lead + (W,), dtype=vt, device="cuda")
    lmg.layer_norm(x, w, b, dense, None, 1e-5, na)
    plain.assert_near(dense, *N.forward())

    dx, check = guarded(lead + (W,), vt, pad, offset)
    dw, check_w = guarded((1, W), pt)
    db, check_b = guarded((1, W), pt)
    lmg.layer_norm_backward(x, w, stats, diff, dx, dw[0], db[0], na)
    want, tol = N.backward(diff)
    for got, v, t in zip((dx, dw[0], db[0]), want, tol):
        plain.assert_near(got, v, t)
    check(), check_w(), check_b()
    again = [guarded(lead + (W,), vt, pad, offset)[0].fill_(3.0)] + [torch.full_like(v, 3.0) for v in (dw[0], db[0])]
    lmg.layer_norm_backward(x, w, stats, diff, *again, na)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw[0], db[0]), again))
    dense = torch.empty(lead + (W,), dtype=vt, device="cuda")
    lmg.layer_norm_backward(x, w, stats, diff, dense, None, None, na)
    plain.assert_near(dense, want[0], tol[0])
    # one of the sums alone, none of them, and in place
    for mask in ((1, 0), (0, 1), (0, 0)):
        got, _ = guarded(lead + (W,), vt, pad, offset)
        alone = [torch.empty(W, dtype=pt, device="cuda") if m else None for m in mask]
        lmg.layer_norm_backward(x, w, stats, diff, got, *alone, na)
        assert torch.equal(got, dx)
        assert all(v is None or torch.equal(v, u[0]) for v, u in zip(alone, (dw, db)))
    lmg.layer_norm_backward(x, w, stats, diff, diff, None, None, na)
    assert torch.equal(diff, dx)
    lmg.layer_norm(x, w, b, x, None, 1e-5, na)
    assert torch.equal(x, out)


def test_layer_norm_of_constant_and_huge_rows():
    """A row without variance is its bias; a row far from zero keeps the digits its values have."""
    W = 48
    x = torch.empty(4, W, device="cuda")
    x[0], x[1] = 3.0, 0.0
    x[2] = 1e4 + torch.arange(W, device="cuda")
    x[3] = float("inf")
    b = torch.arange(W, device="cuda", dtype=F)
    out, stats = torch.empty_like(x), torch.empty(4, 2, device="cuda")
    lmg.layer_norm(x, None, b, out, stats)
    assert torch.equal(out[0], b) and torch.equal(out[1], b) and bool(out[3].isnan().all())
    N = plain.Norm(x[:3], None, b, 1e-5, None)
    want, tol = N.forward()
    plain.assert_near(out[2], want[2], tol[2])
    dx = torch.empty(3, W, device="cuda")
    diff = normal(gen(), 3, W)
    lmg.layer_norm_backward(x[:3], None, stats[:3], diff, dx)
    want, tol = N.backward(diff)
    plain.assert_near(dx, want[0], tol[0])


DROPS = [((1,), F, 0, 0), ((7, 1), F, 0, 0), ((40, 32), F, 0, 0), ((1000, 28), F, 0, 0), ((17, 91, 45), H, 0, 0), ((301, 333), B, 0, 0),
         ((301, 333), F, 3, 1), ((64, 100), H, 4, 4), ((64, 96), B, 8, 0), ((100003,), F, 0, 0), ((100003,), B, 0, 1), ((3, 5000), H, 0, 0),
         ((600, 1024), F, 0, 0)]


@pytest.mark.parametrize("p", [0.0, 1e-4, 0.1, 0.5, 0.99, 1.0])
@pytest.mark.parametrize("shape,dtype,pad,offset", DROPS, ids=["%s-%s-%d" % ("x".join(map(str, c[0])), str(c[1])[6:], c[2]) for c in DROPS])
def test_dropout(shape, dtype, pad, offset, p):
    x = strided(normal(gen(), *shape, dtype=dtype), pad, offset)
    out, check = guarded(shape, dtype, pad, offset)
    lmg.dropout(x, out, p, RNG)
    W = shape[-1]
    f = plain.factors(x.numel() // W, W, p, RNG).view(shape)
    want = x.double() * f
    plain.assert_near(out, want, 2.1 * plain.U * want.abs())
    assert bool(((out == 0) == ((f == 0) | (x == 0))).all())   # a value that stays grows: it is not rounded to zero
    check()
    state = torch.tensor([RNG[0] - (1 << 64), RNG[1]], device="cuda")
    again = torch.empty_like(out)
    lmg.dropout(x, again, p, state)
    assert torch.equal(again, out)
    lmg.dropout(x, x, p, RNG)
    assert torch.equal(x, out)


def test_ties_are_decided_by_the_lower_half():
    """A probability whose upper half meets draws, at whose lower half some of them stay and some fall."""
    rows, W = 4096, 64
    d = plain.draws(rows, W, RNG)
    upper = int(d[100, 5]) >> 16
    p = (upper * 65536 + 32768) / 2.0 ** 32
    tied = (d // 65536) == upper
    assert tied.sum() >= 1
    x = torch.ones(rows, W, device="cuda")
    lmg.dropout(x, x, p, RNG)
    assert torch.equal(x.cpu() != 0, torch.from_numpy(d >= upper * 65536 + 32768))


def test_draws_differ_by_seed_offset_row_and_column():
    x = torch.ones(64, 64, device="cuda")
    outs = []
    for rng in ((1, 0), (2, 0), (1, 1), (1, 1 << 32), (1 << 32, 0)):
        outs.append(torch.empty_like(x))
        lmg.dropout(x, outs[-1], 0.5, rng)
    for i, a in enumerate(outs):
        for b in outs[:i]:
            assert 0.4 < float((a == b).float().mean()) < 0.6
    a = outs[0]
    assert 0.35 < float((a[1:] == a[:-1]).float().mean()) < 0.65 and 0.35 < float((a[:, 8:] == a[:, :-8]).float().mean()) < 0.65


def test_offsets_beyond_31_bits():
    """Rows whose elements lie more than 2^31 from the first."""
    W, R = 32768 + 8, 66000
    types = torch.zeros(R, dtype=torch.int32, device="cuda")
    types[-3:] = torch.tensor([1, -1, 2])
    table = normal(gen(), 3, W, dtype=B)
    out = torch.empty(R, W, dtype=B, device="cuda")
    lmg.embed_types(types, table, out)
    assert torch.equal(out[-3], table[1]) and torch.equal(out[-1], table[2]) and not out[-2].any() and torch.equal(out[7], table[0])
    lmg.dropout(out, out, 0.5, RNG)
    keep = torch.from_numpy(plain.draws(4, W, RNG, first=R - 4) >= 2.0 ** 31).cuda()
    assert torch.equal(out[-4] != 0, keep[0] & (table[0] != 0)) and torch.equal(out[-1], torch.where(keep[3], table[2] * 2, 0))
    lmg.layer_norm(out, None, None, out)
    want, tol = plain.Norm(torch.where(keep[3], table[2] * 2, 0)[None], None, None, 1e-5, None).forward()
    plain.assert_near(out[-1], want[0], tol[0])
    del out
    big, small = torch.zeros(R, W, dtype=B, device="cuda"), normal(gen(), 5, W, dtype=B)
    lmg.embed_types_backward(torch.tensor([0, R - 1, 3, R - 1, R - 2], device="cuda"), small, big)
    assert torch.equal(big[R - 1], (small[1].float() + small[3].float()).to(B)) and torch.equal(big[R - 2], small[4])
    assert not big[4].any() and torch.equal(big[0], small[0])


@pytest.mark.parametrize("lead", [(0,), (0, 4), (4, 0)])
def test_nothing_to_do(lead):
    V, W = 3, 6
    types = torch.zeros(lead, device="cuda")
    na = torch.zeros(lead[0], dtype=torch.int32, device="cuda") if len(lead) == 2 else None
    x = torch.zeros(lead + (W,), device="cuda")
    lmg.embed_types(types, torch.ones(V, W, device="cuda"), x, n_atoms=na)
    grad = torch.full((V, W), GUARD, device="cuda")
    lmg.embed_types_backward(types, x, grad, n_atoms=na)
    assert not grad.any()
    lmg.layer_norm(x, None, None, x, torch.zeros(lead + (2,), device="cuda"), n_atoms=na)
    dw, db = torch.full((W,), GUARD, device="cuda"), torch.full((W,), GUARD, device="cuda")
    lmg.layer_norm_backward(x, None, torch.zeros(lead + (2,), device="cuda"), x, x, dw, db, na)
    assert not dw.any() and not db.any()
    lmg.dropout(x, x, 0.5, RNG)
    # no types, no columns
    out = torch.full((4, W), GUARD, device="cuda")
    lmg.embed_types(torch.zeros(4, device="cuda"), torch.zeros(0, W, device="cuda"), out)
    assert not out.any()
    lmg.embed_types_backward(torch.zeros(4, device="cuda"), out, torch.zeros(0, W, device="cuda"))
    lmg.embed_types(torch.zeros(4, device="cuda"), torch.zeros(3, 0, device="cuda"), torch.zeros(4, 0, device="cuda"))
    lmg.dropout(torch.zeros(4, 0, device="cuda"), torch.zeros(4, 0, device="cuda"), 0.5, RNG)


def test_refusals():
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    ok = (z(4), z(3, 8), z(4, 8))
    for args, kw in [((z(4, dtype=torch.int16),) + ok[1:], {}), ((z(8)[::2],) + ok[1:], {}), ((ok[0], z(3, 8, dtype=torch.float64), ok[2]), {}),
                     ((ok[0], ok[1], z(4, 9)), {}), ((ok[0], ok[1], z(5, 8)), {}), ((ok[0], ok[1], z(8, 4).T), {}),
                     ((ok[0], z(3, 8, dtype=H), ok[2]), {}), ((ok[0], ok[1], z(1, 8).expand(4, 8)), {}),
                     (ok, dict(n_atoms=z(4, dtype=torch.int32))), (ok, dict(p=1.5, rng=RNG)), (ok, dict(p=-0.5, rng=RNG)), (ok, dict(p=0.5)),
                     (ok, dict(p=0.5, rng=(1, 1 << 63))), (ok, dict(p=0.5, rng=(-1, 0))), (ok, dict(p=0.5, rng=(1, 2, 3))),
                     (ok, dict(p=0.5, rng=z(2))), (ok, dict(p=0.5, rng=torch.zeros(2, dtype=torch.int64))), (ok, dict(status=z(1)))]:
        with pytest.raises(ValueError):
            lmg.embed_types(*args, **kw)
    with pytest.raises(TypeError):
        lmg.embed_types([0, 1], ok[1], ok[2])
    with pytest.raises(TypeError):
        lmg.embed_types(ok[0], z(24), ok[2])
    batch = (z(2, 4), z(3, 8), z(2, 4, 8))
    for na in (z(3, dtype=torch.int32), z(2, 2, dtype=torch.int32)):
        with pytest.raises(ValueError):
            lmg.embed_types(*batch, n_atoms=na)
    with pytest.raises(ValueError):
        lmg.embed_types(*(z(2, 8)[:, ::2], z(3, 8), z(2, 4, 8)))
    with pytest.raises(ValueError):   # rows of the batch's examples not evenly spaced
        lmg.embed_types(z(2, 4), z(3, 8), z(2, 5, 8)[:, :4])
    with pytest.raises(ValueError):
        lmg.embed_types_backward(ok[0], z(4, 8, dtype=H), z(3, 8, dtype=B))
    x = z(4, 8)
    for args in [(x, z(7), None, x), (x, z(8, dtype=H), None, x), (x, z(8), z(8, dtype=B), x), (x, None, None, z(4, 9)), (x, None, None, x, z(4, 3)),
                 (x, None, None, x, z(4, 2, dtype=H)), (x, None, None, x, None, 0.0), (x, None, None, x, None, -1.0),
                 (x, None, None, x, None, 1e-5, z(4, dtype=torch.int32)), (x, z(16)[::2], None, x)]:
        with pytest.raises(ValueError):
            lmg.layer_norm(*args)
    h = z(4, 8, dtype=H)
    with pytest.raises(ValueError):
        lmg.layer_norm(h, z(8, dtype=H), z(8), h)
    for args in [(x, None, None, x, x), (x, None, z(4, 2), h, x), (x, None, z(4, 2), x, h), (x, None, z(4, 2), x, x, z(9))]:
        with pytest.raises((ValueError, TypeError)):
            lmg.layer_norm_backward(*args)
    with pytest.raises(ValueError):
        lmg.dropout(x, h, 0.5, RNG)
    with pytest.raises(ValueError):
        lmg.next_draw(torch.zeros(2, dtype=torch.int64))
    nested = torch.nested.nested_tensor([torch.rand(2, 8, device="cuda"), torch.rand(3, 8, device="cuda")])
    with pytest.raises((RuntimeError, TypeError, ValueError)):
        lmg.dropout(nested, nested, 0.5, RNG)
    with pytest.raises((RuntimeError, TypeError, ValueError)):
        torch.vmap(lambda v: lmg.dropout(v, v, 0.5, RNG) or v)(z(3, 4, 8))
    torch.cuda.synchronize()


def test_arrays_on_the_host():
    """Host tensors, numpy arrays and MGrids are staged around the call."""
    g = gen(9)
    types, table = torch.tensor([0., 2, 1, -1]), normal(g, 3, 5)
    want = torch.empty(4, 5, device="cuda")
    lmg.embed_types(types.cuda(), table, want, 2.0, p=0.5, rng=RNG)
    out = torch.empty(4, 5)
    lmg.embed_types(types, table.cpu(), out, 2.0, p=0.5, rng=RNG)
    assert torch.equal(out, want.cpu())
    arr = torch.empty(4, 5).numpy()
    lmg.embed_types(types.numpy(), table.cpu().numpy(), arr, 2.0, p=0.5, rng=RNG)
    assert (arr == want.cpu().numpy()).all()
    m = lmg.MGrid1f(4)
    for i in range(4):
        m[i] = float(types[i])
    lmg.embed_types(m, table, want, 2.0, p=0.5, rng=RNG)
    assert (arr == want.cpu().numpy()).all()
    stats, y, dx, dw = torch.empty(4, 2), torch.empty(4, 5), torch.empty(4, 5), torch.empty(5)
    lmg.layer_norm(out, None, None, y, stats)
    lmg.layer_norm_backward(out, None, stats, out, dx, dw)
    dev = [torch.empty(4, 2, device="cuda"), torch.empty(4, 5, device="cuda"), torch.empty(4, 5, device="cuda"), torch.empty(5, device="cuda")]
    lmg.layer_norm(want, None, None, dev[1], dev[0])
    lmg.layer_norm_backward(want, None, dev[0], want, dev[2], dev[3])
    for a, b in zip((stats, y, dx, dw), dev):
        assert torch.equal(a, b.cpu())


def test_the_general_route_gives_the_same(monkeypatch):
    def everything():
        g = gen(2)
        types, table, na = make_types(g, (3, 50), 9, F), normal(g, 9, 20), torch.tensor([50, 0, 7], device="cuda", dtype=torch.int32)
        x, w = normal(g, 3, 50, 20), normal(g, 20)
        out, grad, y, dx = torch.empty(3, 50, 20, device="cuda"), torch.empty_like(table), torch.empty_like(x), torch.empty_like(x)
        stats, dw, db, z = torch.empty(3, 50, 2, device="cuda"), torch.empty_like(w), torch.empty_like(w), torch.empty_like(x)
        lmg.embed_types(types, table, out, 2.0, na, 0.5, RNG)
        lmg.embed_types_backward(types, x, grad, 2.0, na, 0.5, RNG)
        lmg.layer_norm(x, w, w, y, stats, 1e-3, na)
        lmg.layer_norm_backward(x, w, stats, out, dx, dw, db, na)
        lmg.dropout(x, z, 0.5, RNG)
        return out, grad, y, stats, dx, dw, db, z
    everything()
    from libmolgrid_b200 import molgrid_native as m
    for name in ("_fast_embed", "_fast_embed_backward", "_fast_layer_norm", "_fast_layer_norm_backward", "_fast_dropout"):
        real = getattr(m, name)

        def served(*a, real=real, name=name):
            r = real(*a)
            assert r is not None, name + " left a call on resident tensors to the general route"
            return r
        monkeypatch.setattr(m, name, served)
    fast = everything()
    monkeypatch.setattr(api, "_native", False)
    assert all(torch.equal(a, b) for a, b in zip(fast, everything()))


# ---- modules ----------------------------------------------------------------------------------------------------------
def vectors_64(types, table, weight, bias, eps, scale, n_atoms, f):
    """dropout(layer_norm(scale * table[type])) in 64 bits, its leaves given."""
    rows = table * scale
    if weight is not None:
        rows = (rows - rows.mean(-1, keepdim=True)) / (rows.var(-1, correction=0, keepdim=True) + eps).sqrt() * weight + bias
    t = plain.valid_types(types, table.shape[0], n_atoms)
    return torch.where(t[..., None] >= 0, rows[t.clamp(min=0)], torch.zeros((), dtype=torch.float64, device="cuda")) * f


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_module_and_its_gradients(norm, p):
    """Against differentiation in 64 bits, and the table's gradient against central differences there."""
    g = gen(11)
    B, N, V, W = 3, 60, 7, 12
    types, na = make_types(g, (B, N), V, F), torch.tensor([60, 0, 31], device="cuda", dtype=torch.int32)
    types[2, 40:] = 1e9
    m = lmg.TypeVectors(V, W, scale=3.0, norm=norm, p=p, seed=77, device="cuda")
    if norm:
        m.weight.data += 0.2 * normal(g, W)
        m.bias.data += normal(g, W)
    out = m(types, na)
    f = plain.factors(B * N, W, p, (77, 0)).view(B, N, W)
    leaves = [v.detach().double().requires_grad_() for v in m.parameters()]
    want = vectors_64(types, leaves[0], leaves[1] if norm else None, leaves[2] if norm else None, 1e-5, 3.0, na, f)
    torch.testing.assert_close(out.double(), want, rtol=3e-6, atol=1e-6)   # a norm of 12 values: some 30 roundings of 2^-24
    up = normal(g, B, N, W)
    out.backward(up)
    grads = torch.autograd.grad(want, leaves, up.double())
    for v, w in zip(m.parameters(), grads):
        # sums of up to 91 terms: 100 roundings of the sum of their sizes, some ten times their sum here
        torch.testing.assert_close(v.grad.double(), w, rtol=6e-5, atol=6e-5)
    step = torch.randn(V, W, generator=g, device="cuda", dtype=torch.float64)
    with torch.no_grad():
        ends = [(vectors_64(types, leaves[0] + s * step, leaves[1] if norm else None, leaves[2] if norm else None, 1e-5, 3.0, na, f)
                 * up.double()).sum() for s in (1e-5, -1e-5)]
    assert float((m.table.grad.double() * step).sum()) == pytest.approx(float((ends[0] - ends[1]) / 2e-5), rel=1e-3, abs=1e-3)
    m.check_types()
    types[0, 0] = V
    m(types, na)
    with pytest.raises(IndexError):
        m.check_types()
    m.check_types()
    m.eval()
    assert torch.equal(m(types, na), m(types, na))


def test_half_vectors_of_a_float32_table():
    g = gen(12)
    types = make_types(g, (500,), 20, torch.int64)
    m = lmg.TypeVectors(20, 48, dtype=B, device="cuda", seed=1)
    full = lmg.TypeVectors(20, 48, device="cuda", seed=1)
    full.load_state_dict(m.state_dict())
    out = m(types)
    assert out.dtype is B and torch.equal(out, full(types).to(B))
    up = normal(g, 500, 48, dtype=B)
    out.backward(up)
    full(types).backward(up.float())
    assert m.table.grad.dtype is F
    torch.testing.assert_close(m.table.grad, full.table.grad, rtol=1e-5, atol=1e-5)


def test_lookup_and_dropout_are_differentiable_twice():
    g = gen(13)
    types = make_types(g, (50,), 6, torch.int32)
    table = normal(g, 6, 10).requires_grad_()
    out = lmg.EmbedTypesFunction.apply(types, table, F, 2.0, None, 0.4, RNG, None)
    out = lmg.DropoutFunction.apply(out, 0.2, (5, 6))
    up = normal(g, 50, 10).requires_grad_()
    gt, = torch.autograd.grad(out, table, up, create_graph=True)
    v = normal(g, 6, 10)
    gu, = torch.autograd.grad(gt, up, v)
    f = plain.factors(50, 10, 0.4, RNG) * plain.factors(50, 10, 0.2, (5, 6))
    want = torch.cat([v.double(), torch.zeros(1, 10, device="cuda", dtype=torch.float64)])[plain.valid_types(types, 6, None)] * 2 * f
    torch.testing.assert_close(gu.double(), want, rtol=1e-6, atol=0)
    x = normal(g, 4, 8).requires_grad_()
    y = lmg.LayerNormFunction.apply(x, None, None, 1e-5, None)
    gx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


def test_norm_module_against_64_bits():
    g = gen(14)
    x = normal(g, 3, 20, 33).requires_grad_()
    na = torch.tensor([20, 3, 0], device="cuda", dtype=torch.int32)
    m = lmg.LayerNorm(33, device="cuda")
    m.weight.data += normal(g, 33)
    out = m(x, na)
    up = normal(g, 3, 20, 33)
    out.backward(up.expand(3, 20, 33))
    N = plain.Norm(x.detach(), m.weight.detach(), m.bias.detach(), 1e-5, na)
    plain.assert_near(out.detach(), *N.forward())
    want, tol = N.backward(up)
    for got, v, t in zip((x.grad, m.weight.grad, m.bias.grad), want, tol):
        plain.assert_near(got, v, t)
    x.grad = None
    m(x).sum().backward()                     # a gradient that is one number everywhere
    assert torch.isfinite(x.grad).all()
    with pytest.raises(ValueError):
        m(x[..., :32])


def test_vectors_to_grids():
    """Type indices of a padded batch through Coords2Grid: grids of the atoms alone, gradients back to the table."""
    g = gen(15)
    B, N, V, C = 3, 40, 9, 6
    gm = lmg.GridMaker(0.5, 7.5)
    coords = (torch.rand(B, N, 3, generator=g, device="cuda") - 0.5) * 6
    radii = torch.rand(B, N, generator=g, device="cuda") + 1.0
    types, na = make_types(g, (B, N), V, F), torch.tensor([40, 0, 13], device="cuda", dtype=torch.int32)
    types[2, 13:] = float("nan")              # what a fresh batch holds behind its atoms
    m = lmg.TypeVectors(V, C, p=0.2, seed=3, device="cuda")
    c2g = lmg.Coords2Grid(gm, types=m)
    assert [n for n, _ in c2g.named_parameters()] == ["types.table", "types.weight", "types.bias"]
    grid = c2g(coords, types, radii, na)
    up = normal(g, *grid.shape)
    grid.backward(up)
    vectors = vectors_64(types, m.table.detach().double(), m.weight.detach().double(), m.bias.detach().double(), 1e-5, 1.0, na,
                         plain.factors(B * N, C, 0.2, (3, 0)).view(B, N, C)).float().requires_grad_()
    for b in range(B):
        n = int(na[b])
        want = torch.zeros(gm.grid_dimensions(C), device="cuda")
        if n:
            gm.forward((0, 0, 0), coords[b, :n].contiguous(), vectors[b, :n].detach().contiguous(), radii[b, :n].contiguous(), want)
        torch.testing.assert_close(grid[b], want, rtol=1e-4, atol=1e-5)
    lmg.Coords2Grid(gm)(coords, vectors, radii).backward(up)
    leaves = [v.detach().double().requires_grad_() for v in m.parameters()]
    out = vectors_64(types, *leaves, 1e-5, 1.0, na, plain.factors(B * N, C, 0.2, (3, 0)).view(B, N, C))
    for v, w in zip(m.parameters(), torch.autograd.grad(out, leaves, vectors.grad.double())):
        torch.testing.assert_close(v.grad.double(), w, rtol=2e-4, atol=2e-4 * float(w.abs().max()))
    single = c2g.eval()(coords[0], types[0], radii[0])
    assert single.shape == gm.grid_dimensions(C) and bool(torch.isfinite(single).all())


# ---- streams, graphs, two calls at once -------------------------------------------------------------------------------
def step_inputs(seed, rows=6000, V=900, W=40):
    g = gen(seed)
    types = make_types(g, (rows,), V, torch.int32)
    return types, normal(g, V, W), normal(g, rows, W), torch.empty(V, W, device="cuda"), torch.empty(rows, W, device="cuda")


def whole_step(types, table, diff, grad, out):
    lmg.embed_types(types, table, out, p=0.2, rng=RNG)
    lmg.embed_types_backward(types, diff, grad, p=0.2, rng=RNG)
    stats, dw = torch.empty(table.shape[0], 2, device="cuda"), torch.empty(table.shape[1], device="cuda")
    y, dx = torch.empty_like(table), torch.empty_like(table)
    lmg.layer_norm(table, None, None, y, stats)
    lmg.layer_norm_backward(table, None, stats, grad, dx, dw)
    return out, grad, y, dx, dw


def test_two_streams_at_once():
    a, b = step_inputs(21), step_inputs(22)
    want = [[t.clone() for t in whole_step(*s)] for s in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, st in zip((a, b), streams):
            with torch.cuda.stream(st):
                s[3].fill_(9.0)
                got.append(whole_step(*s))
        torch.cuda.synchronize()
        for w, r in zip(want, got):
            assert all(torch.equal(p, q) for p, q in zip(w, r))


def test_captured_and_replayed():
    """Two graphs, replayed in turn and then together, on inputs that change between replays."""
    sets = [step_inputs(31), step_inputs(32)]
    other = [step_inputs(33), step_inputs(34)]
    for s in sets:
        whole_step(*s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(whole_step(*s))
        graphs.append(g)
    for new in (None, other):
        if new:
            for s, o in zip(sets, new):
                for k in range(3):
                    s[k].copy_(o[k])
        want = [[t.clone() for t in whole_step(s[0], s[1], s[2], torch.empty_like(s[3]), torch.empty_like(s[4]))] for s in sets]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for w, r in zip(want, outs):
            assert all(torch.equal(p, q) for p, q in zip(w, r))


def test_replays_take_draws_of_their_own():
    m = lmg.Dropout(0.5, seed=4, device="cuda")
    x = torch.ones(32, 40, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        m(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = m(x)
    seen = []
    for k in range(3):
        g.replay()
        torch.cuda.synchronize()
        seen.append(y.clone())
        assert torch.equal(y != 0, plain.factors(32, 40, 0.5, (4, 1 + k)) != 0)
    assert m.generator.tolist() == [4, 4]
    assert not torch.equal(seen[0], seen[1])


def test_training_step_captured():
    """Forward and backward of the module in one graph; no eager graph of its leaves lives meanwhile."""
    g = gen(41)
    types, up = make_types(g, (2000,), 30, F), normal(g, 2000, 16)
    m = lmg.TypeVectors(30, 16, p=0.1, seed=9, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m(types).backward(up)
    torch.cuda.current_stream().wait_stream(side)
    for v in m.parameters():
        v.grad = None
    gc.collect()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m(types).backward(up)
    for k in (1, 2):
        graph.replay()
        torch.cuda.synchronize()
        twin = lmg.TypeVectors(30, 16, p=0.1, seed=9, device="cuda")
        twin.load_state_dict(m.state_dict())
        twin.generator[1] = k
        twin(types).backward(up)
        for v, w in zip(m.parameters(), twin.parameters()):
            assert torch.equal(v.grad, w.grad)


def test_launches_are_counted():
    lib = _cabi.lib()
    s = step_inputs(51)
    n = lib.lmg_launch_count()
    lmg.embed_types(s[0], s[1], s[4])
    assert lib.lmg_launch_count() == n + 1
    lmg.embed_types_backward(s[0], s[2], s[3])
    assert lib.lmg_launch_count() > n + 1
