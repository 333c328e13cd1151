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
