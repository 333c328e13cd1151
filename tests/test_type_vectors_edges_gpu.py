"""Learned type vectors on the GPU at the ends of their ranges, and beside the calls that they are used with."""
import pytest
import torch

import libmolgrid_b200 as lmg
from tests import vectors_plain as plain
from tests.test_type_vectors_gpu import gen, guarded, normal, strided

pytestmark = pytest.mark.gpu

F, B, H = torch.float32, torch.bfloat16, torch.float16


# ---- a few wide rows that do not begin on 16 bytes --------------------------------------------------------------------
@pytest.mark.parametrize("vt,pt", [(F, F), (B, F), (H, H)], ids=["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("W", [505, 506, 509, 510, 511, 512, 513, 1001, 2049, 8185])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5])
def test_norm_of_few_wide_rows(rows, W, vt, pt):
    g = gen(rows * 10000 + W)
    for pad, offset in ((0, 0), (1, 0), (0, 1)):
        x, diff = strided(normal(g, rows, W, dtype=vt), pad, offset), strided(normal(g, rows, W, dtype=vt), pad, offset)
        w, b = (1 + 0.3 * normal(g, W)).to(pt), normal(g, W).to(pt)
        out, check = guarded((rows, W), vt, pad, offset)
        stats = torch.empty(rows, 2, device="cuda")
        lmg.layer_norm(x, w, b, out, stats)
        N = plain.Norm(x, w, b, 1e-5, None)
        plain.assert_near(out, *N.forward())
        check()
        want, tol = N.backward(diff)
        dx, check = guarded((rows, W), vt, pad, offset)
        dw, db = torch.empty(W, dtype=pt, device="cuda"), torch.empty(W, dtype=pt, device="cuda")
        lmg.layer_norm_backward(x, w, stats, diff, dx, dw, db)
        for got, v, t in zip((dx, dw, db), want, tol):
            plain.assert_near(got, v, t)
        check()
        alone, check = guarded((rows, W), vt, pad, offset)
        lmg.layer_norm_backward(x, w, stats, diff, alone)
        assert torch.equal(alone, dx)
        check()


def test_norm_modules_of_few_wide_rows():
    g = gen(2)
    m = lmg.LayerNorm(1001, device="cuda")
    x = normal(g, 3, 1001).requires_grad_()
    up = normal(g, 3, 1001)
    m(x).backward(up)
    want, tol = plain.Norm(x.detach(), m.weight.detach(), m.bias.detach(), 1e-5, None).backward(up)
    for got, v, t in zip((x.grad, m.weight.grad, m.bias.grad), want, tol):
        plain.assert_near(got, v, t)
    m = lmg.TypeVectors(3, 1001, device="cuda", seed=5)
    m(torch.tensor([0, 2, 1, 2], device="cuda")).backward(normal(g, 4, 1001))
    assert all(bool(torch.isfinite(v.grad).all()) for v in m.parameters())


# ---- what GridMaker.check_types reads ---------------------------------------------------------------------------------
GRADIENTS = [
    # slots, types, width: few types, many types (one cluster sorts; several launches)
    ("tables", lambda: table_gradient(20000, 28, 28)), ("sort", lambda: table_gradient(20000, 5000, 64)),
    ("long sort", lambda: table_gradient(40000, 5000, 24)), ("norm", lambda: norm_gradient(3000, 28)), ("wide norm", lambda: norm_gradient(200, 8200)),
    ("small", lambda: table_gradient(500, 5000, 24)),
]


def table_gradient(n, V, W):
    g = gen(5)
    types = torch.randint(0, V, (n,), generator=g, device="cuda", dtype=torch.int32)
    lmg.embed_types_backward(types, normal(g, n, W), torch.empty(V, W, device="cuda"))


def norm_gradient(n, W):
    g = gen(5)
    x = normal(g, n, W)
    out, stats, dw = torch.empty_like(x), torch.empty(n, 2, device="cuda"), torch.empty(W, device="cuda")
    lmg.layer_norm(x, None, None, out, stats)
    lmg.layer_norm_backward(x, None, stats, out, torch.empty_like(x), dw, torch.empty_like(dw))


@pytest.mark.parametrize("native", [True, False], ids=["compiled", "general"])
@pytest.mark.parametrize("gradient", [c[1] for c in GRADIENTS], ids=[c[0] for c in GRADIENTS])
def test_gradients_leave_what_check_types_reads(gradient, native, monkeypatch):
    from libmolgrid_b200 import api
    if not native:
        monkeypatch.setattr(api, "_native", False)
    g = gen(1)
    gm = lmg.GridMaker(0.5, 7.5)
    n, C = 3000, 4
    coords, radii = (torch.rand(n, 3, generator=g, device="cuda") - 0.5) * 6, torch.ones(n, device="cuda")
    grid = torch.empty(gm.grid_dimensions(C), device="cuda")
    good = torch.randint(0, C, (n,), generator=g, device="cuda").float()
    bad = good.clone()
    bad[1234] = C
    for _ in range(2):     # the second time with buffers that there are already
        gm.forward((0, 0, 0), coords, good, radii, grid)
        gradient()
        gm.check_types()
        gm.forward((0, 0, 0), coords, bad, radii, grid)
        gradient()
        with pytest.raises(IndexError):
            gm.check_types()


def test_training_step_leaves_what_check_types_reads():
    g = gen(3)
    B, N, V, C = 4, 2000, 28, 6
    gm = lmg.GridMaker(0.5, 7.5)
    m = lmg.TypeVectors(V, C, seed=3, device="cuda")
    c2g = lmg.Coords2Grid(gm, types=m)
    coords, radii = (torch.rand(B, N, 3, generator=g, device="cuda") - 0.5) * 6, torch.ones(B, N, device="cuda")
    types = torch.randint(0, V, (B, N), generator=g, device="cuda").float()
    for _ in range(2):
        out = c2g(coords, types, radii)
        out.backward(normal(g, *out.shape))
        gm.check_types()
        m.check_types()


@pytest.mark.parametrize("n,V,W", [(20000, 28, 28), (20000, 5000, 64), (40000, 5000, 24)])
def test_a_workspace_that_a_gradient_took_has_no_status(n, V, W):
    """At the C interface one workspace may serve both: what a gradient wrote over is not read as a gridding call's flags."""
    import ctypes
    from libmolgrid_b200 import _cabi, api
    lib = _cabi.lib()
    g = gen(7)
    gm = lmg.GridMaker(0.5, 7.5)
    types = torch.randint(0, V, (n,), generator=g, device="cuda").float()
    coords, radii = (torch.rand(n, 3, generator=g, device="cuda") - 0.5) * 6, torch.ones(n, device="cuda")
    gm.forward((0, 0, 0), coords, types, radii, torch.empty(gm.grid_dimensions(4), device="cuda"))   # types beyond the channels
    ws, st = gm._last_ws, api._stream_ptr(torch.device("cuda", torch.cuda.current_device()))
    assert lib.lmg_check_status(ctypes.c_void_p(ws.data_ptr()), st) == _cabi.LMG_ERR_OUT_OF_RANGE
    big = torch.empty(lib.lmg_vectors_workspace_bytes(_cabi.OP_EMBED_BACKWARD, n, V, W) + ws.numel(), dtype=torch.uint8, device="cuda")
    big[:ws.numel()] = ws
    s = _cabi.SlotsStruct()
    s.batch, s.max_atoms, s.type_index, s.index_type = 1, n, types.data_ptr(), _cabi.INDEX_FLOAT32
    diff, grad = normal(g, n, W), torch.empty(V, W, device="cuda")
    vec = [_cabi.VectorsStruct(t.data_ptr(), _cabi.FLOAT32, W) for t in (diff, grad)]
    _cabi.check(lib.lmg_embed_types_backward(ctypes.byref(s), V, W, ctypes.byref(vec[0]), 1.0, None, ctypes.byref(vec[1]),
                                             ctypes.c_void_p(big.data_ptr()), big.numel(), st))
    assert lib.lmg_check_status(ctypes.c_void_p(big.data_ptr()), st) == _cabi.LMG_OK


# ---- passes that are computed again -----------------------------------------------------------------------------------
def gradients(m, call, up):
    for v in m.parameters():
        v.grad = None
    out = call()
    out.backward(up)
    return [out.detach()] + [v.grad.clone() for v in m.parameters()]


@pytest.mark.parametrize("reentrant", [True, False])
def test_a_checkpointed_module_has_the_same_gradients(reentrant):
    from torch.utils.checkpoint import checkpoint
    g = gen(8)
    V, W, n = 20, 16, 500
    types = torch.randint(0, V, (n,), generator=g, device="cuda")
    m = torch.nn.Sequential(lmg.TypeVectors(V, W, p=0.3, seed=3, device="cuda"), lmg.Dropout(0.4, seed=4, device="cuda"))
    vectors, drop = m
    up, leaf = normal(g, n, W), torch.zeros((), device="cuda", requires_grad=True)   # a reentrant pass wants an input with a gradient
    a, b = vectors.draw(), drop.draw()
    assert a.tolist() == [3, 0] and vectors.generator.tolist() == [3, 1]

    def forward(z):
        return drop(vectors(types, draw=a), draw=b) + z
    want = gradients(m, lambda: forward(leaf), up)
    got = gradients(m, lambda: checkpoint(forward, leaf, use_reentrant=reentrant), up)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    assert vectors.generator.tolist() == [3, 1] and drop.generator.tolist() == [4, 1]
    # without a draw the pass would take others the second time
    for again in (lambda z: vectors(types) + z, lambda z: drop(vectors(types, draw=a)) + z):
        out = checkpoint(again, leaf, use_reentrant=reentrant)
        with pytest.raises(RuntimeError, match="draw"):
            out.backward(up)
    m.eval()
    want = gradients(m, lambda: drop(vectors(types)) + leaf, up)
    got = gradients(m, lambda: checkpoint(lambda z: drop(vectors(types)) + z, leaf, use_reentrant=reentrant), up)
    assert all(torch.equal(p, q) for p, q in zip(want, got)) and vectors.draw() is None


def test_a_given_draw():
    m = lmg.Dropout(0.5, seed=9, device="cuda")
    x = torch.ones(40, 24, device="cuda")
    first = m(x)                                             # draw 0 of its own
    assert torch.equal(m(x, draw=(9, 0)), first) and m.generator.tolist() == [9, 1]
    assert torch.equal(m(x, draw=torch.tensor([9, 0], device="cuda")), first)
    assert torch.equal(m.eval()(x, draw=(9, 0)), x)
    with pytest.raises(ValueError):
        m.train()(x, draw=(9, 1 << 63))


def test_types_to_grids_computed_again():
    from torch.utils.checkpoint import checkpoint
    g = gen(10)
    B, N, V, C = 2, 30, 9, 5
    gm = lmg.GridMaker(0.5, 7.5)
    m = lmg.TypeVectors(V, C, p=0.4, seed=3, device="cuda")
    c2g = lmg.Coords2Grid(gm, types=m)
    coords = ((torch.rand(B, N, 3, generator=g, device="cuda") - 0.5) * 6).requires_grad_()
    radii, types = torch.ones(B, N, device="cuda"), torch.randint(0, V, (B, N), generator=g, device="cuda").float()
    na, draw = torch.tensor([30, 11], dtype=torch.int32, device="cuda"), m.draw()
    up = normal(g, B, *gm.grid_dimensions(C))
    want = gradients(m, lambda: c2g(coords, types, radii, na, draw=draw), up)
    got = gradients(m, lambda: checkpoint(lambda c: c2g(c, types, radii, na, draw=draw), coords, use_reentrant=False), up)
    # densities and gradients of atoms are summed in an order that varies; the table's are not
    for p, q in zip(want, got):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-5)
    with pytest.raises(ValueError):
        lmg.Coords2Grid(gm)(coords, torch.zeros(B, N, C, device="cuda"), radii, draw=draw)


# ---- the widest rows --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("W", [65535 * 1024, 65535 * 1024 + 4, 65535 * 1024 + 1, 1 << 26, (1 << 26) + 4])
def test_the_widest_rows(W):
    table = torch.arange(W, device="cuda", dtype=F)[None]
    out = torch.full((2, W), 5.0, device="cuda")
    lmg.embed_types(torch.tensor([0, -1], device="cuda"), table, out, 2.0)
    assert torch.equal(out[0], table[0] * 2) and not out[1].any()
    lmg.dropout(out, out, 0.0, (1, 0))
    assert torch.equal(out[0], table[0] * 2)
    lmg.dropout(table, out[:1], 0.5, (1, 0))
    kept = torch.from_numpy(plain.draws(1, 4096, (1, 0)) >= 2.0 ** 31).cuda()
    assert torch.equal(out[0, 1:4096] != 0, kept[0, 1:])
    stays = out[0] != 0
    assert torch.equal(out[0][stays], table[0][stays] * 2) and abs(float(stays.double().mean()) - 0.5) < 5 * 0.5 / W ** 0.5


# ---- more slots than 2^30 ---------------------------------------------------------------------------------------------
def test_gradient_of_more_than_a_billion_slots():
    from libmolgrid_b200 import _cabi, api
    R, V = (1 << 30) + 5, 100000      # 17 bits of keys, two a pass: nine passes of two launches, the sums and what crosses their blocks
    types = torch.arange(R, device="cuda", dtype=torch.int32).remainder_(V)
    diff = types.remainder(7).add_(1).to(B)[:, None]
    grad = torch.full((V, 1), 5.0, device="cuda")
    n = _cabi.lib().lmg_launch_count()
    lmg.embed_types_backward(types, diff, grad)
    launches = _cabi.lib().lmg_launch_count() - n
    t = torch.arange(V, device="cuda")
    slots = R // V + (t < R % V)
    assert torch.equal(grad[:, 0].double(), slots.double() * (t % 7 + 1))     # whole numbers below 2^24: exact in any order
    assert launches == 20
    api._other_workspaces.clear()
    del types, diff
    torch.cuda.empty_cache()


# ---- padded batches to grids ------------------------------------------------------------------------------------------
class Shifted(torch.nn.Module):
    """Vectors with something added to all of them, empty slots too."""

    def __init__(self, V, C):
        super().__init__()
        self.vectors, self.shift = lmg.TypeVectors(V, C, seed=1, device="cuda"), torch.nn.Parameter(torch.full((C,), 0.7, device="cuda"))

    def forward(self, types, n_atoms=None):
        return self.vectors(types, n_atoms) + self.shift


@pytest.mark.parametrize("maker", ["python", "compiled"])
@pytest.mark.parametrize("counts", ["list", "int32", "int64"])
def test_padding_is_not_gridded(maker, counts):
    if maker == "python":
        gm = lmg.GridMaker(0.5, 7.5)
    else:
        import molgrid
        gm = molgrid.GridMaker(0.5, 7.5)
    g = gen(16)
    B, N, V, C = 4, 40, 9, 6
    na = [40, 0, 13, 1]
    coords = (torch.rand(B, N, 3, generator=g, device="cuda") - 0.5) * 6
    radii = torch.rand(B, N, generator=g, device="cuda") + 1.0
    types = torch.randint(0, V, (B, N), generator=g, device="cuda").float()
    m = Shifted(V, C)
    up = normal(g, B, *gm.grid_dimensions(C))
    want = []
    for b, n in enumerate(na):
        c = coords[b, :n].clone().requires_grad_()
        out = lmg.Coords2Grid(gm, types=m)(c, types[b, :n], radii[b, :n])
        out.backward(up[b])
        want.append((out.detach(), c.grad))
    shift = m.shift.grad.clone()
    for fill in (None, float("nan"), 1e30, float("inf")):
        if fill is not None:
            for b, n in enumerate(na):
                coords[b, n:], radii[b, n:], types[b, n:] = fill, fill, fill
        for v in m.parameters():
            v.grad = None
        c = coords.clone().requires_grad_()
        counted = na if counts == "list" else torch.tensor(na, dtype=getattr(torch, counts), device="cuda")
        out = lmg.Coords2Grid(gm, types=m)(c, types, radii, counted)
        out.backward(up)
        for b, n in enumerate(na):
            # sums of up to 40 densities and of some thousand voxels, whose order goes by the batch
            torch.testing.assert_close(out[b], want[b][0], rtol=1e-5, atol=1e-5)
            torch.testing.assert_close(c.grad[b, :n], want[b][1], rtol=1e-4, atol=1e-3)
            assert not c.grad[b, n:].any()
        torch.testing.assert_close(m.shift.grad, shift, rtol=1e-4, atol=1e-2)


@pytest.mark.parametrize("by_type", [False, True], ids=["radii by atom", "radii by type"])
@pytest.mark.parametrize("maker", ["python", "compiled"])
def test_padding_and_second_derivatives(maker, by_type):
    import molgrid
    g = gen(17)
    B, N, V, C = 3, 20, 9, 4
    gm = (lmg if maker == "python" else molgrid).GridMaker(0.5, 7.5, False, by_type)
    na = [20, 0, 7]
    coords = (torch.rand(B, N, 3, generator=g, device="cuda") - 0.5) * 6
    radii, types = torch.ones(B, C if by_type else N, device="cuda"), torch.randint(0, V, (B, N), generator=g, device="cuda").float()
    m = Shifted(V, C)
    up, v = normal(g, B, *gm.grid_dimensions(C)), normal(g, B, N, 3)

    def forces(b, n, c, counted):
        out = lmg.Coords2Grid(gm, types=m)(c, types if counted else types[b, :n], radii if counted else radii[b] if by_type else radii[b, :n],
                                           *([counted] if counted else []))
        up_ = (up if counted else up[b]).clone().requires_grad_()
        f, = torch.autograd.grad(out, c, up_, create_graph=True)
        return torch.autograd.grad(f, [up_, m.shift], v if counted else v[b, :n], retain_graph=False)

    one = [forces(b, n, coords[b, :n].clone().requires_grad_(), None) for b, n in enumerate(na) if n]
    for b, n in enumerate(na):
        coords[b, n:] = float("nan")
        if not by_type:
            radii[b, n:] = float("nan")
    all_up, all_shift = forces(0, 0, coords.clone().requires_grad_(), na)
    for (u, _), b in zip(one, (0, 2)):
        torch.testing.assert_close(all_up[b], u, rtol=1e-4, atol=1e-3)
    assert not all_up[1].any()
    torch.testing.assert_close(all_shift, one[0][1] + one[1][1], rtol=1e-4, atol=1e-2)


def test_counts_without_a_batch():
    gm, m = lmg.GridMaker(0.5, 7.5), Shifted(3, 4)
    with pytest.raises(ValueError):
        lmg.Coords2Grid(gm, types=m)(torch.zeros(5, 3, device="cuda"), torch.zeros(5, device="cuda"), torch.ones(5, device="cuda"), [5])


# ---- the ends of the ranges of a table --------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,V,W,p", [(5, 3, 1 << 20, 0.3), (5, 3, (1 << 20) + 8, 0.3), (7, 2, 1 << 23, 0.0), (1100, 40, 70001, 0.2)])
def test_gradients_of_wide_tables(rows, V, W, p):
    g = gen(W)
    types = torch.randint(-1, V, (rows,), generator=g, device="cuda", dtype=torch.int32)
    diff = normal(g, rows, W, dtype=H)
    grad, check = guarded((V, W), F)
    lmg.embed_types_backward(types, diff, grad, 0.5, p=p, rng=(3, 4))
    plain.assert_near(grad, *plain.embed_backward(types, diff, V, 0.5, None, p, (3, 4)))
    check()


def test_the_most_types():
    """2^31 - 1 rows of one value: keys of 31 bits, and addresses beyond them."""
    V = (1 << 31) - 1
    table = torch.zeros(V, 1, dtype=B, device="cuda")
    some = torch.tensor([0, 1, V - 1, 1 << 30, V - 2, 12345678], device="cuda")
    table[some, 0] = torch.arange(1, 7, device="cuda").to(B)
    types = some.repeat(500)
    types[7] = V                                   # beyond the table
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.empty(types.shape[0], 1, dtype=B, device="cuda")
    lmg.embed_types(types, table, out, status=status)
    want = torch.arange(1, 7, device="cuda").repeat(500)
    want[7] = 0
    assert torch.equal(out[:, 0].long(), want) and int(status) == 1
    table.fill_(3.0)
    lmg.embed_types_backward(types, torch.ones_like(out), table)
    assert table[some, 0].tolist() == [500] * 6    # 499 of the second: halfway between 498 and 500, whose last bit of eight is even
    table[some] = 0
    assert not bool(table.view(torch.int16).any())
    for kind in (torch.int32, F):                  # what float32 holds: 2^31 - 1 is no number of it
        few = torch.tensor([1 << 30, 5, -1], device="cuda").to(kind)
        lmg.embed_types_backward(few.repeat(600), torch.ones(1800, 1, dtype=B, device="cuda"), table)
        assert table[[1 << 30, 5, 0], 0].tolist() == [600, 600, 0]
        table[[1 << 30, 5]] = 0
        assert not bool(table.view(torch.int16).any())
    del table
    torch.cuda.empty_cache()


def test_gradients_into_rows_with_gaps_beyond_4_gb():
    g = gen(23)
    V, W, rows = 70000, 32768, 1100
    grad, check = guarded((V, W), B, 8)
    types = torch.randint(0, V, (rows,), generator=g, device="cuda")
    types[-40:] = torch.tensor([V - 1, 3], device="cuda").repeat(20)
    diff = normal(g, rows, W, dtype=B)
    grad.fill_(9.0)
    lmg.embed_types_backward(types, diff, grad)
    check()
    met = types.unique()
    rank = torch.searchsorted(met, types)
    want, tol = plain.embed_backward(rank, diff, met.numel(), 1.0, None, 0.0, None)
    plain.assert_near(grad[met], want, tol)
    grad[met] = 0
    assert not bool(grad.view(V, W).any())
    del grad, check
    torch.cuda.empty_cache()


def test_rows_with_gaps_captured():
    """A table's gradient that is cleared before the sort, in a graph."""
    g = gen(24)
    V, W, rows = 5000, 24, 9000
    types, diff = torch.randint(0, V, (rows,), generator=g, device="cuda"), normal(g, rows, W)
    grad, check = guarded((V, W), F, 4)
    lmg.embed_types_backward(types, diff, grad)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lmg.embed_types_backward(types, diff, grad)
    for seed in (25, 26):
        types.copy_(torch.randint(0, V, (rows,), generator=gen(seed), device="cuda"))
        grad.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        plain.assert_near(grad, *plain.embed_backward(types, diff, V, 1.0, None, 0.0, None))
        check()


# ---- batches assembled on the GPU -------------------------------------------------------------------------------------
def test_types_of_a_device_batch(tmp_path):
    import numpy as np
    from libmolgrid_b200 import coord_cache
    rng = np.random.default_rng(3)
    lines = []
    for i in range(4):
        for name, n in (("r%d.gninatypes" % i, int(rng.integers(20, 90))), ("l%d.gninatypes" % i, int(rng.integers(3, 30)))):
            coord_cache.write_gninatypes(tmp_path / name, rng.normal(size=(n, 3)) * 3, rng.integers(0, 30, n))
        lines.append("1 0.5 r%d.gninatypes l%d.gninatypes" % (i, i))
    (tmp_path / "list.types").write_text("\n".join(lines) + "\n")
    p = coord_cache.ExampleProvider(data_root=str(tmp_path))
    p.populate(str(tmp_path / "list.types"))
    batch = p.next_device_batch(4)
    batch.check()
    V, W = batch.num_types(), 6
    types, na = batch.type_index, batch.n_atoms
    g = gen(4)
    table = normal(g, V, W)
    out, again = (torch.full(tuple(types.shape) + (W,), 5.0, device="cuda") for _ in range(2))
    lmg.embed_types(batch, table, out)
    lmg.embed_types(types, table, again, n_atoms=na)
    assert torch.equal(out, again)
    plain.assert_near(out, *plain.embed(types, table, 1.0, na, 0.0, None))
    up, grad, want = normal(g, *out.shape), torch.empty_like(table), torch.empty_like(table)
    lmg.embed_types_backward(batch, up, grad)
    lmg.embed_types_backward(types, up, want, n_atoms=na)
    assert torch.equal(grad, want)
    m = lmg.TypeVectors(V, W, device="cuda", seed=1)
    assert torch.equal(m(batch), m(types, na))
    for call in (lambda: lmg.embed_types(batch, table, out, n_atoms=na), lambda: m(batch, na)):
        with pytest.raises(TypeError):
            call()
    c2g = lmg.Coords2Grid(lmg.GridMaker(0.5, 7.5), types=m)
    grids = c2g(batch.coords, types, batch.radii, na)
    grids.sum().backward()
    assert bool(torch.isfinite(grids).all()) and all(bool(torch.isfinite(v.grad).all()) for v in m.parameters())
    m.check_types()


# ---- threads ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("own_streams", [True, False])
def test_threads_at_once(own_streams):
    """Calls of four threads, whose scratch differs in size and lies under way together."""
    import threading
    g = gen(30)
    inputs, want = [], []
    for k, (n, V, W) in enumerate([(20000, 28, 28), (20000, 5000, 64), (40000, 5000, 24), (9000, 60, 300)]):
        types, x = torch.randint(0, V, (n,), generator=g, device="cuda"), normal(g, n, W)
        inputs.append((types, x, V))

    def step(types, x, V):
        grad, out, stats = torch.empty(V, x.shape[1], device="cuda"), torch.empty_like(x), torch.empty(x.shape[0], 2, device="cuda")
        dw, dx = torch.empty(x.shape[1], device="cuda"), torch.empty_like(x)
        lmg.embed_types_backward(types, x, grad)
        lmg.layer_norm(x, None, None, out, stats)
        lmg.layer_norm_backward(x, None, stats, out, dx, dw)
        return grad, out, dx, dw
    want = [step(*i) for i in inputs]
    torch.cuda.synchronize()
    failures = []

    def work(k):
        stream = torch.cuda.Stream() if own_streams else torch.cuda.current_stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = step(*inputs[k])
                stream.synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, want[k])):
                    failures.append(k)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
