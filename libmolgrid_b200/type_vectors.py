"""Learned type vectors: what a network makes of atom types before they are gridded.

The functions fill caller-provided arrays, as ``GridMaker.forward`` does: ``embed_types`` looks type indices up in a
table, ``layer_norm`` normalises rows, ``dropout`` drops values by a counter-based generator whose masks are made again
in the backward pass instead of being stored, and ``embed_types_backward`` / ``layer_norm_backward`` give the gradients.
``TypeVectors`` is the module of all three, and what ``Coords2Grid(..., types=...)`` calls on type indices.

Vectors are float32, bfloat16 or float16 with the values of a row next to each other; rows may lie further apart than
they are long (a slice of wider rows).  Type indices are float32 (what the example provider hands out), int32 or int64.
A slot is empty where its type is negative and, with ``n_atoms``, behind its example's atom count; what lies there is not
read.  Empty slots get zero vectors, which carry no weight in a grid, and have no part in any gradient.  The reference has
no counterpart: a type vector is an input there (include/libmolgrid/coordinateset.h:30-39).
"""
import ctypes

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from . import _cabi
from . import api as _api
from . import grids as _grids
from ._cabi import check
from .api import _Arg, _current_device, _fast, _other_workspaces, _stream_ptr, _workspace

_VECTORS = {torch.float32: _cabi.FLOAT32, torch.bfloat16: _cabi.BFLOAT16, torch.float16: _cabi.FLOAT16}
_INDICES = {torch.float32: _cabi.INDEX_FLOAT32, torch.int32: _cabi.INDEX_INT32, torch.int64: _cabi.INDEX_INT64}


class _Typed(object):
    """An array argument of one of ``dtypes`` on the GPU for the duration of one call."""

    def __init__(self, obj, device, name, dtypes, output=False):
        obj = _grids.operand_tensor(obj)
        if isinstance(obj, np.ndarray):
            obj = torch.from_numpy(obj)
        elif not torch.is_tensor(obj):
            raise TypeError("%s: expected a Grid, MGrid, torch tensor or numpy array" % name)
        if obj.dtype not in dtypes:
            raise ValueError("%s: %s is none of %s" % (name, obj.dtype, ", ".join(str(d) for d in dtypes)))
        self.host = None
        if obj.is_cuda:
            if obj.device != device:
                raise ValueError("%s: tensor on %s but current device is %s" % (name, obj.device, device))
            self.t = obj
        else:
            self.host = obj
            self.t = _Arg._stage(obj, device, output)
        self.type, self.output = dtypes[obj.dtype], output

    def finish(self):
        if self.output and self.host is not None:
            self.host.copy_(self.t)


def _row_stride(t, name):
    """Elements from one row of t to the next, all rows taken in order."""
    shape, strides = t.shape, t.stride()
    if shape[-1] > 1 and strides[-1] != 1:
        raise ValueError("%s: the values of a row are not next to each other" % name)
    ld = None
    for n, s in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if n == 1:
            continue
        if ld is None:
            ld, step = s, s * n
        elif s != step:
            raise ValueError("%s: rows are not evenly spaced" % name)
        else:
            step *= n
    if ld is None:
        return max(1, int(shape[-1]))
    if ld < shape[-1]:
        raise ValueError("%s: rows overlap" % name)
    return int(ld)


class _Vectors(_Typed):
    """Rows of vectors."""

    def __init__(self, obj, device, name, output=False):
        _Typed.__init__(self, obj, device, name, _VECTORS, output)
        if self.t.dim() < 1:
            raise TypeError("%s: expected rows" % name)
        if max(self.t.shape[-1], self.t.shape[0]) >= 1 << 31:
            raise ValueError("%s: 2^31 rows or columns and more" % name)
        ld = 1 if self.t.numel() == 0 else _row_stride(self.t, name)
        self.struct = _cabi.VectorsStruct(self.t.data_ptr(), self.type, max(ld, int(self.t.shape[-1])))

    def shaped(self, shape, name):
        if tuple(self.t.shape) != tuple(shape):
            raise ValueError("%s: expected shape %s, got %s" % (name, tuple(shape), tuple(self.t.shape)))
        return self


def _dense(obj, device, name, dtypes, shape, output=False):
    a = _Typed(obj, device, name, dtypes, output)
    if tuple(a.t.shape) != tuple(shape):
        raise ValueError("%s: expected shape %s, got %s" % (name, tuple(shape), tuple(a.t.shape)))
    if not a.t.is_contiguous():
        raise ValueError("%s: tensor is not contiguous" % name)
    return a


def _slots(lead, n_atoms, device):
    """(struct, what it points to) of the slots of an array with these leading dimensions."""
    s, keep = _cabi.SlotsStruct(), []
    if n_atoms is None:
        n = 1
        for d in lead:
            n *= int(d)
        s.batch, s.max_atoms = 1, n
        if n >= 1 << 31:
            raise ValueError("2^31 slots and more")
        return s, keep
    if len(lead) != 2:
        raise ValueError("n_atoms goes with batches: slots of shape (batch, atoms)")
    if int(lead[0]) * int(lead[1]) >= 1 << 31:
        raise ValueError("2^31 slots and more")
    s.batch, s.max_atoms = int(lead[0]), int(lead[1])
    na = torch.as_tensor(n_atoms).to(device=device, dtype=torch.int32).contiguous()
    if tuple(na.shape) != (s.batch,):
        raise ValueError("n_atoms must have one entry per example")
    keep.append(na)
    s.n_atoms = na.data_ptr()
    return s, keep


def _types(types, n_atoms, device, status):
    """The slots of type indices (or of a DeviceBatch, which brings its own counts)."""
    from .coord_cache import DeviceBatch
    if isinstance(types, DeviceBatch):
        if n_atoms is not None:
            raise TypeError("a DeviceBatch has atom counts of its own")
        types, n_atoms = types.type_index, types.n_atoms
    t = _Typed(types, device, "types", _INDICES)
    if not t.t.is_contiguous():
        raise ValueError("types: tensor is not contiguous")
    s, keep = _slots(t.t.shape, n_atoms, device)
    s.type_index, s.index_type = t.t.data_ptr(), t.type
    keep.append(t)
    if status is not None:
        if not (torch.is_tensor(status) and status.is_cuda and status.dtype is torch.int32 and status.numel() == 1):
            raise ValueError("status: expected one int32 on the GPU")
        if status.device != device:
            raise ValueError("status: tensor on %s but current device is %s" % (status.device, device))
        keep.append(status)
        s.status = status.data_ptr()
    return t.t, s, keep


def _drop(p, rng, device):
    """The struct of a dropout, None where nothing is dropped."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout probability outside [0, 1]")
    if p == 0.0:
        return None
    if torch.is_tensor(rng):
        if rng.dtype is not torch.int64 or not rng.is_cuda or tuple(rng.shape) != (2,) or not rng.is_contiguous():
            raise ValueError("rng: expected a seed and an offset, or two int64 on the GPU")
        if rng.device != device:
            raise ValueError("rng: tensor on %s but current device is %s" % (rng.device, device))
        return _cabi.DropoutStruct(p, 0, 0, rng.data_ptr())
    if rng is None or len(rng) != 2:
        raise ValueError("rng: expected a seed and an offset, or two int64 on the GPU")
    seed, offset = int(rng[0]), int(rng[1])
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 63):
        raise ValueError("rng: seeds are whole numbers below 2^64, offsets below 2^63")
    return _cabi.DropoutStruct(p, seed, offset, None)


def _ref(s):
    return None if s is None else ctypes.byref(s)


# Each call goes to the compiled module first, which serves it when every array is a CUDA tensor of the right kind and shape, and
# answers None when not: the general route takes those (and raises what there is to raise).
def embed_types(types, table, out, scale=1.0, n_atoms=None, p=0.0, rng=None, status=None):
    """``out[slot] = scale * table[types[slot]]``, then dropout with probability ``p``; empty slots are zero.

    ``types`` (N,) or (B,N) - or a ``DeviceBatch`` -, ``table`` (ntypes,W), ``out`` types' shape + (W,).  A float32
    table may have 16-bit outputs; otherwise the two types agree.  ``rng`` is (seed, offset), or an int64 CUDA tensor of the two, which
    the kernel reads: see :func:`dropout`.  A type >= ntypes leaves its slot empty and sets ``status``, one int32 on
    the GPU that the caller clears and reads when it suits (the check that ``GridMaker.check_types`` makes)."""
    m = _api._native or _fast()
    if m and m._fast_embed(types, table, out, scale, n_atoms, p, rng, status) is not None:
        return
    dev = _current_device()
    t, s, keep = _types(types, n_atoms, dev, status)
    tab = _Vectors(table, dev, "table")
    if tab.t.dim() != 2:
        raise TypeError("table: expected 2 dimensions, got %d" % tab.t.dim())
    o = _Vectors(out, dev, "out", output=True).shaped(tuple(t.shape) + (tab.t.shape[1],), "out")
    drop = _drop(p, rng, dev)
    check(_cabi.lib().lmg_embed_types(ctypes.byref(s), int(tab.t.shape[0]), int(tab.t.shape[1]), ctypes.byref(tab.struct),
                                      float(scale), _ref(drop), ctypes.byref(o.struct), _stream_ptr(dev)))
    o.finish()


def embed_types_backward(types, diff, table_gradients, scale=1.0, n_atoms=None, p=0.0, rng=None, status=None):
    """``table_gradients[type] = scale * sum of diff[slot]`` over the type's slots, ``diff`` after the same dropout as the
    vectors; types without a slot get zero.  16-bit gradients may go into a float32 table."""
    m = _api._native or _fast()
    if m and m._fast_embed_backward(types, diff, table_gradients, scale, n_atoms, p, rng,
            status, _other_workspaces.by) is not None:
        return
    dev = _current_device()
    t, s, keep = _types(types, n_atoms, dev, status)
    g = _Vectors(table_gradients, dev, "table_gradients", output=True)
    if g.t.dim() != 2:
        raise TypeError("table_gradients: expected 2 dimensions, got %d" % g.t.dim())
    V, W = int(g.t.shape[0]), int(g.t.shape[1])
    d = _Vectors(diff, dev, "diff").shaped(tuple(t.shape) + (W,), "diff")
    drop = _drop(p, rng, dev)
    ws = _workspace(dev, _cabi.lib().lmg_vectors_workspace_bytes(_cabi.OP_EMBED_BACKWARD, s.batch * s.max_atoms, V, W), kept=_other_workspaces)
    check(_cabi.lib().lmg_embed_types_backward(ctypes.byref(s), V, W, ctypes.byref(d.struct), float(scale), _ref(drop),
                                               ctypes.byref(g.struct), ctypes.c_void_p(ws.data_ptr()), ws.numel(),
                                               _stream_ptr(dev)))
    g.finish()


def _parameter(w, device, name, vectors, output=False):
    """One value a column, float32 or of the vectors' type, or None."""
    if w is None:
        return None
    return _dense(w, device, name, {torch.float32: _cabi.FLOAT32, vectors.t.dtype: vectors.type}, (vectors.t.shape[-1],), output)


def _parameter_type(*parameters):
    """The common element type of those that there are."""
    types = {a.type for a in parameters if a is not None}
    if len(types) > 1:
        raise ValueError("weights, biases and their gradients differ in type")
    return types.pop() if types else _cabi.FLOAT32


def _data(a):
    return None if a is None else ctypes.c_void_p(a.t.data_ptr())


def layer_norm(x, weight, bias, out, stats=None, eps=1e-5, n_atoms=None):
    """``out = (x - mean) / sqrt(variance + eps) * weight + bias`` over the last dimension.

    ``x`` and ``out`` (...,W) of one type (``out`` may be ``x``), ``weight`` and ``bias`` (W,) of that type or float32, or None.
    ``n_atoms`` (B,) goes with ``x`` (B,N,W): rows behind an example's count become zero.  ``stats`` (...,2)
    float32 takes each row's mean and 1 / sqrt(variance + eps), which the backward pass reads."""
    m = _api._native or _fast()
    if m and m._fast_layer_norm(x, weight, bias, out, stats, eps, n_atoms) is not None:
        return
    dev = _current_device()
    a = _Vectors(x, dev, "x")
    o = _Vectors(out, dev, "out", output=True).shaped(a.t.shape, "out")
    w, b = _parameter(weight, dev, "weight", a), _parameter(bias, dev, "bias", a)
    wtype = _parameter_type(w, b)
    st = None if stats is None else _dense(stats, dev, "stats", {torch.float32: 0}, tuple(a.t.shape[:-1]) + (2,), True)
    s, keep = _slots(a.t.shape[:-1], n_atoms, dev)
    check(_cabi.lib().lmg_layer_norm(ctypes.byref(s), int(a.t.shape[-1]), ctypes.byref(a.struct), _data(w), _data(b), wtype,
                                     float(eps), ctypes.byref(o.struct), _data(st), _stream_ptr(dev)))
    o.finish()
    if st is not None:
        st.finish()


def layer_norm_backward(x, weight, stats, diff, x_gradients, weight_gradients=None, bias_gradients=None, n_atoms=None):
    """Gradients of :func:`layer_norm` from ``diff``, that of its output, and the ``stats`` it filled.  ``x_gradients`` may
    be ``diff``; gradients of weights or biases that are not wanted are None."""
    m = _api._native or _fast()
    if m and m._fast_layer_norm_backward(x, weight, stats, diff, x_gradients, weight_gradients,
            bias_gradients, n_atoms, _other_workspaces.by) is not None:
        return
    dev = _current_device()
    a = _Vectors(x, dev, "x")
    d = _Vectors(diff, dev, "diff").shaped(a.t.shape, "diff")
    g = _Vectors(x_gradients, dev, "x_gradients", output=True).shaped(a.t.shape, "x_gradients")
    w = _parameter(weight, dev, "weight", a)
    dw = _parameter(weight_gradients, dev, "weight_gradients", a, True)
    db = _parameter(bias_gradients, dev, "bias_gradients", a, True)
    wtype = _parameter_type(w, dw, db)
    st = _dense(stats, dev, "stats", {torch.float32: 0}, tuple(a.t.shape[:-1]) + (2,))
    s, keep = _slots(a.t.shape[:-1], n_atoms, dev)
    W = int(a.t.shape[-1])
    ws = _workspace(dev, _cabi.lib().lmg_vectors_workspace_bytes(_cabi.OP_LAYER_NORM_BACKWARD, s.batch * s.max_atoms, 0, W),
                    kept=_other_workspaces)
    check(_cabi.lib().lmg_layer_norm_backward(ctypes.byref(s), W, ctypes.byref(a.struct), _data(w), wtype, _data(st),
                                              ctypes.byref(d.struct), ctypes.byref(g.struct), _data(dw), _data(db),
                                              ctypes.c_void_p(ws.data_ptr()), ws.numel(), _stream_ptr(dev)))
    for r in (g, dw, db):
        if r is not None:
            r.finish()


def dropout(x, out, p, rng):
    """``out = x / (1 - p)`` where a value stays and 0 where it is dropped, with probability ``p``.

    ``x`` and ``out`` (...,W) of one type; ``out`` may be ``x``.  Which values stay goes by the seed, the offset, a value's
    row (all leading dimensions taken in order) and its column alone, so the gradient is the same call on the gradient.
    ``rng`` is (seed, offset) - another offset for each draw - or an int64 CUDA tensor of the two, which the kernel reads
    (:func:`next_draw` takes it from a generator state on the GPU: the form for calls that are captured and replayed)."""
    m = _api._native or _fast()
    if m and m._fast_dropout(x, out, p, rng) is not None:
        return
    dev = _current_device()
    a = _Vectors(x, dev, "x")
    o = _Vectors(out, dev, "out", output=True).shaped(a.t.shape, "out")
    drop = _drop(p, rng, dev) or _cabi.DropoutStruct(0.0, 0, 0, None)
    s, _ = _slots(a.t.shape[:-1], None, dev)
    check(_cabi.lib().lmg_dropout(s.max_atoms, int(a.t.shape[-1]), ctypes.byref(a.struct), ctypes.byref(drop),
                                  ctypes.byref(o.struct), _stream_ptr(dev)))
    o.finish()


def generator_state(seed, device=None):
    """A generator on the GPU: its seed and the offset of its next draw, as two int64."""
    seed = int(seed)
    if not 0 <= seed < 1 << 64:
        raise ValueError("rng: seeds are whole numbers below 2^64")
    return torch.tensor([seed - (1 << 64) if seed >> 63 else seed, 0], dtype=torch.int64, device=device or _current_device())


def next_draw(state):
    """One draw of a generator on the GPU, as :func:`dropout` takes it; the state moves on by one, at every replay too
    where the call is captured."""
    dev = _current_device()
    if not (torch.is_tensor(state) and state.is_cuda and state.dtype is torch.int64 and tuple(state.shape) == (2,)
            and state.is_contiguous()):
        raise ValueError("state: expected two int64 on the GPU")
    if state.device != dev:
        raise ValueError("state: tensor on %s but current device is %s" % (state.device, dev))
    taken = torch.empty_like(state)
    check(_cabi.lib().lmg_dropout_next(ctypes.c_void_p(state.data_ptr()), ctypes.c_void_p(taken.data_ptr()), _stream_ptr(dev)))
    return taken


# ------------------------------------------------------------------------------------------------
# autograd
# ------------------------------------------------------------------------------------------------
def _counts(n_atoms, like):
    """Atom counts as a tensor next to ``like``, as autograd keeps it; None stays."""
    return None if n_atoms is None else torch.as_tensor(n_atoms).to(device=like.device, dtype=torch.int32)


class EmbedTypesGradientFunction(torch.autograd.Function):
    """Gradient of the lookup as a differentiable function of the vectors' gradient."""

    @staticmethod
    def forward(ctx, types, diff, ntypes, dtype, scale, n_atoms, p, rng):
        ctx.save_for_backward(types, n_atoms, rng if torch.is_tensor(rng) else None)
        ctx.settings = (scale, p, None if torch.is_tensor(rng) else rng, diff.dtype)
        grad = torch.empty((ntypes, diff.shape[-1]), dtype=dtype, device=diff.device)
        embed_types_backward(types, diff.contiguous(), grad, scale, n_atoms, p, rng)
        return grad

    @staticmethod
    def backward(ctx, grad):
        types, n_atoms, state = ctx.saved_tensors
        scale, p, rng, dtype = ctx.settings
        dd = EmbedTypesFunction.apply(types, grad, dtype, scale, n_atoms, p, rng if state is None else state, None)
        return None, dd, None, None, None, None, None, None


class EmbedTypesFunction(torch.autograd.Function):
    """types (...), table (ntypes,W) -> vectors (...,W) of ``dtype``; differentiable in the table, any number of times."""

    @staticmethod
    def forward(ctx, types, table, dtype, scale, n_atoms, p, rng, status):
        types, n_atoms = types.contiguous(), _counts(n_atoms, table)
        ctx.save_for_backward(types, n_atoms, rng if torch.is_tensor(rng) else None)
        ctx.settings = (scale, p, None if torch.is_tensor(rng) else rng, table.shape[0], table.dtype)
        out = torch.empty(tuple(types.shape) + (table.shape[1],), dtype=dtype, device=table.device)
        embed_types(types, table.contiguous(), out, scale, n_atoms, p, rng, status)
        return out

    @staticmethod
    def backward(ctx, diff):
        types, n_atoms, state = ctx.saved_tensors
        scale, p, rng, ntypes, dtype = ctx.settings
        grad = EmbedTypesGradientFunction.apply(types, diff, ntypes, dtype, scale, n_atoms, p, rng if state is None else state)
        return None, grad, None, None, None, None, None, None


class LayerNormFunction(torch.autograd.Function):
    """x (...,W), weight and bias (W,) or None -> normalised rows; differentiable once."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, n_atoms):
        x, n_atoms = x.contiguous(), _counts(n_atoms, x)
        out, stats = torch.empty_like(x), torch.empty(tuple(x.shape[:-1]) + (2,), dtype=torch.float32, device=x.device)
        layer_norm(x, weight, bias, out, stats, eps, n_atoms)
        ctx.save_for_backward(x, weight, bias, stats, n_atoms)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, diff):
        x, weight, bias, stats, n_atoms = ctx.saved_tensors
        dx = torch.empty_like(x)
        dw = torch.empty_like(weight) if weight is not None and ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if bias is not None and ctx.needs_input_grad[2] else None
        layer_norm_backward(x, weight, stats, diff.contiguous(), dx, dw, db, n_atoms)
        return dx, dw, db, None, None


class DropoutFunction(torch.autograd.Function):
    """x (...,W) -> x dropped; differentiable any number of times."""

    @staticmethod
    def forward(ctx, x, p, rng):
        ctx.save_for_backward(rng if torch.is_tensor(rng) else None)
        ctx.settings = (p, None if torch.is_tensor(rng) else rng)
        x = x.contiguous()
        out = torch.empty_like(x)
        dropout(x, out, p, rng)
        return out

    @staticmethod
    def backward(ctx, diff):
        state, = ctx.saved_tensors
        p, rng = ctx.settings
        return DropoutFunction.apply(diff, p, rng if state is None else state), None, None


# ------------------------------------------------------------------------------------------------
# modules
# ------------------------------------------------------------------------------------------------
class _Drawing(torch.nn.Module):
    """A module that drops values in training.  Its generator moves with the module to the GPU and with the state dict from run to
    run.  Without ``seed`` torch's host generator gives one.  It is a rank's own and no buffer, which ``DistributedDataParallel`` would
    copy from rank 0: ranks that are to drop different values get different seeds."""

    _ranks_own = ("generator",)   # tensors that move with the module

    def __init__(self, p, seed, device):
        super().__init__()
        self.p = float(p)
        if not 0.0 <= self.p <= 1.0:
            raise ValueError("dropout probability outside [0, 1]")
        seed = int(torch.randint(1 << 62, (1,)).item()) if seed is None else int(seed)
        self.generator = generator_state(seed, device or "cpu")

    def _apply(self, fn, *args, **kw):
        super()._apply(fn, *args, **kw)
        for name in self._ranks_own:
            setattr(self, name, fn(getattr(self, name)))
        return self

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        destination[prefix + "generator"] = self.generator

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        key = prefix + "generator"
        if key in unexpected_keys:
            unexpected_keys.remove(key)
        given = state_dict.get(key)
        if given is None:
            if strict:
                missing_keys.append(key)
        elif not torch.is_tensor(given) or given.dtype is not torch.int64 or tuple(given.shape) != (2,):
            error_msgs.append("%s: expected the seed and the offset of a generator, two int64" % key)
        elif local_metadata.get("assign_to_params_buffers"):
            self.generator = given
        else:
            self.generator.copy_(given)

    def draw(self):
        """One draw of the module's generator, to be given to a call - or to the two of a pass that is computed again in the
        backward pass (``torch.utils.checkpoint``); None where nothing is dropped."""
        return next_draw(self.generator) if self.training and self.p > 0.0 else None

    def _draw(self, given):
        """(p, draw) of this call."""
        if not self.training or self.p == 0.0:
            return 0.0, None
        if given is None:
            if torch._C._current_graph_task_id() != -1:   # a backward pass is under way
                raise RuntimeError("a pass that is computed again would drop other values than the first time: give both the same "
                                   "draw, forward(..., draw=module.draw())")
            given = next_draw(self.generator)
        return self.p, given


class Dropout(_Drawing):
    """Dropout of the last dimension's values while training, without a stored mask.  ``draw`` as :func:`dropout` takes it
    (:meth:`draw`, or a seed and an offset); without it each call takes the generator's next."""

    def __init__(self, p=0.5, seed=None, device=None):
        super().__init__(p, seed, device)

    def forward(self, x, draw=None):
        p, draw = self._draw(draw)
        return x if draw is None else DropoutFunction.apply(x, p, draw)

    def extra_repr(self):
        return "p={}".format(self.p)


class LayerNorm(torch.nn.Module):
    """Layer norm over the last dimension; rows behind ``n_atoms`` of a padded batch become zero."""

    def __init__(self, width, eps=1e-5, device=None, dtype=None):
        super().__init__()
        self.width, self.eps = int(width), float(eps)
        self.weight = torch.nn.Parameter(torch.ones(self.width, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(self.width, device=device, dtype=dtype))

    def forward(self, x, n_atoms=None):
        if x.shape[-1] != self.width:
            raise ValueError("x: expected rows of %d values, got %d" % (self.width, x.shape[-1]))
        return LayerNormFunction.apply(x, self.weight, self.bias, self.eps, n_atoms)

    def extra_repr(self):
        return "{}, eps={}".format(self.width, self.eps)


class TypeVectors(_Drawing):
    """Type indices to learned vectors: ``dropout(layer_norm(scale * table[type]))``, empty slots zero.

    ``TypeVectors(ntypes, width)(types[, n_atoms])`` with ``types`` (N,) or (B,N), or a ``DeviceBatch``.  Every slot of a type
    has the same normalised row, so the table is normalised, not the slots, and the gradients of all slots of a type are
    summed before they go through the norm.  The scale goes into the norm's eps there: layer_norm(s x, eps) is layer_norm(x, eps / s^2).
    A type >= ntypes is an empty slot; :meth:`check_types` raises for it.  ``draw`` as in :class:`Dropout`."""

    _ranks_own = ("generator", "status")

    def __init__(self, ntypes, width, scale=1.0, norm=True, p=0.0, eps=1e-5, seed=None, dtype=torch.float32, device=None):
        super().__init__(p, seed, device)
        self.scale, self.eps, self.dtype = float(scale), float(eps), dtype
        if norm and not self.scale > 0.0:
            raise ValueError("scale must be positive where its result is normalised")
        float32 = torch.finfo(torch.float32)
        if norm and not float32.tiny <= self._norm_eps() <= float32.max:
            raise ValueError("eps / scale^2, the norm's eps on the table itself, is beyond float32")
        if dtype not in _VECTORS:
            raise ValueError("dtype: %s is none of %s" % (dtype, ", ".join(str(d) for d in _VECTORS)))
        self.table = torch.nn.Parameter(torch.randn(int(ntypes), int(width), device=device))
        if norm:
            self.weight = torch.nn.Parameter(torch.ones(int(width), device=device))
            self.bias = torch.nn.Parameter(torch.zeros(int(width), device=device))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)

    def _norm_eps(self):
        square = self.scale * self.scale
        return self.eps / square if square > 0.0 else float("inf")

    def forward(self, types, n_atoms=None, draw=None):
        from .coord_cache import DeviceBatch
        if isinstance(types, DeviceBatch):
            if n_atoms is not None:
                raise TypeError("a DeviceBatch has atom counts of its own")
            types, n_atoms = types.type_index, types.n_atoms
        p, draw = self._draw(draw)
        table, scale = self.table, self.scale
        if self.weight is not None:
            table, scale = LayerNormFunction.apply(table, self.weight, self.bias, self._norm_eps(), None), 1.0
        return EmbedTypesFunction.apply(types, table, self.dtype, scale, n_atoms, p, draw, self.status)

    def check_types(self):
        """Synchronise and raise IndexError if a call since the last check met a type beyond the table."""
        bad = int(self.status.item())
        self.status.zero_()
        if bad:
            raise IndexError("type index beyond the table of %d types" % self.table.shape[0])

    def extra_repr(self):
        return "{}, {}, scale={}, norm={}, p={}".format(self.table.shape[0], self.table.shape[1], self.scale,
                                                        self.weight is not None, self.p)
