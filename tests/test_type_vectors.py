"""Learned type vectors without a GPU: layouts, refusals at the C interface, the generator and the division by multiplication."""
import ctypes
import random

import numpy as np
import pytest
import torch

from libmolgrid_b200 import _cabi
from tests import vectors_plain as plain

P = 1 << 20   # an address that is never followed: the call fails before any launch


def vec(ld, type=_cabi.FLOAT32, data=P):
    return _cabi.VectorsStruct(data, type, ld)


def slots(batch=2, n=3, index=P, kind=_cabi.INDEX_FLOAT32):
    s = _cabi.SlotsStruct()
    s.batch, s.max_atoms, s.type_index, s.index_type = batch, n, index, kind
    return s


def test_struct_layouts(lib):
    assert ctypes.sizeof(_cabi.VectorsStruct) == 24
    assert ctypes.sizeof(_cabi.SlotsStruct) == 4 * 2 + 8 * 2 + 8 + 8
    assert ctypes.sizeof(_cabi.DropoutStruct) == 32


def refused(lib, rc, text, code=_cabi.LMG_ERR_INVALID_ARGUMENT):
    assert rc == code, (rc, lib.lmg_last_error())
    assert text in lib.lmg_last_error().decode()


def test_lookup_refusals(lib):
    def call(s=None, V=5, W=4, table=None, drop=None, out=None):
        return lib.lmg_embed_types(s or slots(), V, W, table or vec(4), 1.0, drop, out or vec(4), None)
    refused(lib, call(slots(-1)), "negative size")
    refused(lib, call(V=-1), "negative size")
    refused(lib, call(W=-4), "negative size")
    refused(lib, call(slots(1 << 16, 1 << 15)), "2^31 slots")
    refused(lib, call(W=1 << 30, table=vec(1 << 30), out=vec(1 << 30)), "2^30 columns")
    refused(lib, call(slots(index=None)), "type indices missing memory")
    refused(lib, call(slots(kind=3)), "unknown element type")
    refused(lib, call(table=vec(3)), "rows overlap")
    refused(lib, call(table=vec(4, 7)), "unknown element type")
    refused(lib, call(out=vec(4, data=None)), "missing memory")
    refused(lib, call(out=vec(4, data=P + 2)), "not aligned")
    refused(lib, call(table=vec(4, _cabi.BFLOAT16)), "differ in type")
    refused(lib, call(table=vec(4, _cabi.BFLOAT16), out=vec(4, _cabi.FLOAT16)), "differ in type")
    for p in (-0.1, 1.1, float("nan")):
        refused(lib, call(drop=_cabi.DropoutStruct(p, 0, 0, None)), "probability")
    refused(lib, call(drop=_cabi.DropoutStruct(0.5, 0, 1 << 63, None)), "offset")
    assert call(slots(0)) == call(slots(2, 0)) == call(W=0) == _cabi.LMG_OK      # nothing to do


def test_gradient_refusals(lib):
    def call(s=None, V=5, W=4, diff=None, grad=None, ws=P, nbytes=1 << 40):
        return lib.lmg_embed_types_backward(s or slots(), V, W, diff or vec(4), 1.0, None, grad or vec(4), ws, nbytes, None)
    refused(lib, call(W=(1 << 23) + 1, diff=vec(1 << 24), grad=vec(1 << 24)), "2^23 columns")
    refused(lib, call(ws=P + 8), "off 16 bytes", _cabi.LMG_ERR_WORKSPACE)
    refused(lib, call(grad=vec(4, _cabi.FLOAT16)), "differ in type")
    refused(lib, call(diff=vec(4, _cabi.FLOAT16), grad=vec(4, _cabi.BFLOAT16)), "differ in type")
    refused(lib, call(ws=None), "workspace too small", _cabi.LMG_ERR_WORKSPACE)
    refused(lib, call(nbytes=8), "workspace too small", _cabi.LMG_ERR_WORKSPACE)
    refused(lib, call(diff=vec(4, data=None)), "missing memory")
    assert call(V=0) == call(W=0) == _cabi.LMG_OK


def test_norm_refusals(lib):
    def call(s=None, W=4, x=None, wtype=_cabi.FLOAT32, eps=1e-5, out=None):
        return lib.lmg_layer_norm(s or slots(), W, x or vec(4), None, None, wtype, eps, out or vec(4), None, None)
    for eps in (0.0, -1.0, float("nan")):
        refused(lib, call(eps=eps), "eps")
    refused(lib, call(x=vec(4, _cabi.FLOAT16)), "differ in type")
    refused(lib, call(wtype=_cabi.FLOAT16), "neither float32")
    refused(lib, call(wtype=9), "neither float32")
    assert call(slots(0)) == call(W=0) == _cabi.LMG_OK

    def back(x=None, stats=P, diff=None, grad=None, wtype=_cabi.FLOAT32, ws=P, nbytes=1 << 40):
        return lib.lmg_layer_norm_backward(slots(), 4, x or vec(4), None, wtype, stats, diff or vec(4), grad or vec(4), None, None, ws,
                                           nbytes, None)
    refused(lib, back(stats=None), "stats missing")
    refused(lib, back(stats=P + 4), "not aligned to 8")
    refused(lib, back(ws=P + 8), "off 16 bytes", _cabi.LMG_ERR_WORKSPACE)
    refused(lib, back(diff=vec(4, _cabi.FLOAT16)), "differ in type")
    refused(lib, back(grad=vec(2)), "rows overlap")
    refused(lib, back(ws=None), "workspace too small", _cabi.LMG_ERR_WORKSPACE)


def test_dropout_refusals(lib):
    d = _cabi.DropoutStruct(0.5, 0, 0, None)
    refused(lib, lib.lmg_dropout(-1, 4, vec(4), d, vec(4), None), "negative size")
    refused(lib, lib.lmg_dropout(2, 4, vec(4), None, vec(4), None), "null dropout")
    refused(lib, lib.lmg_dropout(2, 4, vec(4), d, vec(4, _cabi.FLOAT16), None), "differ in type")
    refused(lib, lib.lmg_dropout(2, 4, vec(4), _cabi.DropoutStruct(2.0, 0, 0, None), vec(4), None), "probability")
    refused(lib, lib.lmg_dropout_next(None, P, None), "missing memory")
    assert lib.lmg_dropout(0, 4, vec(4), d, vec(4), None) == _cabi.LMG_OK


def test_workspaces_are_never_zero(lib):
    for op in (_cabi.OP_EMBED_BACKWARD, _cabi.OP_LAYER_NORM_BACKWARD):
        assert lib.lmg_vectors_workspace_bytes(op, 0, 0, 0) > 0
        assert lib.lmg_vectors_workspace_bytes(op, 4000, 28, 32) >= lib.lmg_vectors_workspace_bytes(op, 0, 28, 32)


def test_generator_known_answers():
    """The published vectors of Philox4x32-10, and the layout of the draws."""
    ones = 0xffffffff
    assert plain.philox([0] * 4, [0] * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert plain.philox([ones] * 4, [ones] * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert plain.philox([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0]) == \
        [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]
    rng = (0x123456789abcdef0, 0x7eadbeefcafef00d)
    d = plain.draws(5, 19, rng, first=3)
    for r, c in ((0, 0), (4, 18), (2, 9), (1, 7)):
        w = [plain.philox([c // 8, 3 + r, rng[1] & ones, rng[1] >> 32 | top], [rng[0] & ones, rng[0] >> 32]) for top in (0, 1 << 31)]
        h = [x[c % 8 // 2] >> 16 * (c % 2) & 0xffff for x in w]
        assert d[r, c] == h[0] * 65536 + h[1]


def test_draws_are_even():
    """A tenth of a million draws fall below a tenth of the range, give or take five deviations."""
    d = plain.draws(1000, 1000, (7, 0))
    share = (d < 0.1 * 2 ** 32).mean()
    assert abs(share - 0.1) < 5 * np.sqrt(0.09 / 1e6)


def test_division_by_multiplication():
    def div(n, d):
        shift = 0
        while shift < 32 and (1 << shift) < d:
            shift += 1
        mul = ((1 << 32) * ((1 << shift) - d) // d + 1) & 0xffffffff
        return ((n * mul >> 32) + n & 0xffffffff) >> shift
    r = random.Random(3)
    for d in [1, 2, 3, 5, 7, 28, 4000, 65535, 65536, (1 << 31) - 1, 1 << 30] + [r.randrange(1, 1 << 31) for _ in range(300)]:
        for n in [0, 1, d - 1, d, min(d + 1, (1 << 31) - 1), (1 << 31) - 1] + [r.randrange(1 << 31) for _ in range(50)]:
            assert div(n, d) == n // d, (n, d)


def test_modules_keep_their_state():
    import libmolgrid_b200 as lmg
    torch.manual_seed(5)
    m = lmg.TypeVectors(14, 6, p=0.25)
    assert {n for n, _ in m.named_parameters()} == {"table", "weight", "bias"}
    assert set(m.state_dict()) == {"table", "weight", "bias", "generator"}
    other = lmg.TypeVectors(14, 6, p=0.25)
    assert not torch.equal(m.generator, other.generator)
    other.load_state_dict(m.state_dict())
    assert torch.equal(m.generator, other.generator)
    assert {n for n, _ in lmg.TypeVectors(3, 2, norm=False).named_parameters()} == {"table"}
    assert lmg.generator_state((1 << 64) - 1, "cpu").tolist() == [-1, 0]
    for bad in (dict(p=1.5), dict(scale=0.0), dict(dtype=torch.float64)):
        with pytest.raises(ValueError):
            lmg.TypeVectors(3, 2, **bad)
    with pytest.raises(ValueError):
        lmg.generator_state(1 << 64, "cpu")
    with pytest.raises(ValueError):
        lmg.Coords2Grid(lmg.GridMaker(0.5, 5.5))(torch.zeros(2, 4, 3), torch.zeros(2, 4, 2), torch.ones(2, 4), torch.zeros(2))


def test_no_cpu_fallback():
    import libmolgrid_b200 as lmg
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(RuntimeError):
        lmg.embed_types(torch.zeros(3), torch.ones(2, 4), torch.zeros(3, 4))
    with pytest.raises(RuntimeError):
        lmg.layer_norm(torch.zeros(3, 4), None, None, torch.zeros(3, 4))
    with pytest.raises(RuntimeError):
        lmg.dropout(torch.zeros(3, 4), torch.zeros(3, 4), 0.5, (1, 0))
