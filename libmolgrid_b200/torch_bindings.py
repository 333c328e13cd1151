"""torch.autograd integration of the gridding path (reference: python/torch_bindings.py:44-162).

``Coords2Grid`` turns coordinates, type vectors and radii into a density grid and is
differentiable with respect to coordinates and types, twice (the second derivative goes through
``GridMaker.backward_gradients``).  Batched input is gridded in one pass over the whole batch;
the reference loops over the batch in Python.
"""
import torch

from .api import GridMaker, float3  # noqa: F401


def _batched(coords):
    return coords.dim() == 3


def _counted(n_atoms):
    return {} if n_atoms is None else {"n_atoms": n_atoms}


class Grid2CoordsGradientFunction(torch.autograd.Function):
    """Backward pass of gridding as a differentiable function of (coords, types, grid gradient)."""

    @staticmethod
    def forward(ctx, gmaker, center, coords, types, radii, grid_gradient, n_atoms=None):
        ctx.save_for_backward(coords, types, radii, grid_gradient, n_atoms)
        ctx.gmaker, ctx.center = gmaker, center
        grad_coords = torch.empty_like(coords)
        grad_types = torch.empty_like(types)
        gmaker.backward(center, coords, types, radii, grid_gradient.contiguous(), grad_coords, grad_types, **_counted(n_atoms))
        return grad_coords, grad_types

    @staticmethod
    def backward(ctx, grad_coords, grad_types):
        coords, types, radii, grid_gradient, n_atoms = ctx.saved_tensors
        ddcoords = torch.empty_like(coords)
        ddtypes = torch.empty_like(types)
        ddgrid = torch.empty_like(grid_gradient)
        ctx.gmaker.backward_gradients(ctx.center, coords, types, radii, grid_gradient.contiguous(),
                                      grad_coords.contiguous(), grad_types.contiguous(), ddgrid, ddcoords, ddtypes,
                                      **_counted(n_atoms))
        return None, None, ddcoords, ddtypes, None, ddgrid, None


class Coords2GridFunction(torch.autograd.Function):
    """coords (N,3) or (B,N,3), vector types (N,T) or (B,N,T), radii (N,)/(T,) or (B,N)/(B,T) -> grid.  ``n_atoms``, int32 on the
    GPU (B,), leaves out what lies behind an example's atoms."""

    @staticmethod
    def forward(ctx, gmaker, center, coords, types, radii, n_atoms=None):
        if types.dim() != coords.dim():
            raise ValueError("Vector types required in Coords2Grid.")
        if _batched(coords) and (coords.shape[0] != types.shape[0] or coords.shape[0] != radii.shape[0]):
            raise RuntimeError("Inconsistent batch sizes in Coords2Grid inputs")
        ctx.save_for_backward(coords, types, radii, n_atoms)
        ctx.gmaker, ctx.center = gmaker, center
        shape = gmaker.grid_dimensions(types.shape[-1])
        if _batched(coords):
            shape = (coords.shape[0],) + shape
        output = torch.empty(shape, dtype=coords.dtype, device=coords.device)
        gmaker.forward(center, coords, types, radii, output, **_counted(n_atoms))
        return output

    @staticmethod
    def backward(ctx, grid_gradient):
        coords, types, radii, n_atoms = ctx.saved_tensors
        if not ctx.needs_input_grad[3] and not torch.is_grad_enabled():
            # types are inputs, not parameters, and no second derivative is being recorded: only the
            # channels in which an atom carries weight need to be read
            grad_coords = torch.empty_like(coords)
            ctx.gmaker.backward_arrays(ctx.center, coords, types, radii, grid_gradient.contiguous(), grad_coords,
                                       want_type_gradients=False, **_counted(n_atoms))
            return None, None, grad_coords, None, None, None
        grad_coords, grad_types = Grid2CoordsGradientFunction.apply(ctx.gmaker, ctx.center, coords, types, radii,
                                                                    grid_gradient, n_atoms)
        return None, None, grad_coords, grad_types, None, None


# the reference has a separate class for batched input; here one function serves both ranks
BatchedCoords2GridFunction = Coords2GridFunction


class Coords2Grid(torch.nn.Module):
    """Module form: ``Coords2Grid(gmaker, center=(0,0,0))(coords, types, radii)``.

    ``types=`` takes a module that makes type vectors of type indices, such as ``TypeVectors(ntypes, channels)``: ``types``
    may then be indices (N,) or (B,N), with ``n_atoms`` (B,) in padded batches, and gradients reach the module's table.  Slots behind an
    example's atoms are not gridded, whatever they hold, and have gradients of zero.  A ``draw`` is handed to that module.  Vectors
    are gridded as float32: those of 16 bits are converted by the caller."""

    def __init__(self, gmaker, center=(0, 0, 0), types=None):
        super().__init__()
        self.gmaker = gmaker
        self.center = center
        self.types = types

    def forward(self, coords, types, radii, n_atoms=None, draw=None):
        if self.types is not None and types.dim() == coords.dim() - 1:
            if n_atoms is not None:
                n_atoms = torch.as_tensor(n_atoms).to(device=coords.device, dtype=torch.int32)
            types = self.types(types, *(() if n_atoms is None else (n_atoms,)), **({} if draw is None else {"draw": draw}))
        elif n_atoms is not None or draw is not None:
            raise ValueError("n_atoms and draw go with type indices that a module turns into vectors")
        coords, types, radii = coords.contiguous(), types.contiguous(), radii.contiguous()
        single = coords.dim() == 2 and types.dim() == 2 and radii.dim() == 1
        batched = coords.dim() == 3 and types.dim() == 3 and radii.dim() == 2
        if not (single or batched):
            raise RuntimeError("Invalid input dimensions in forward of Coords2Grid")
        if n_atoms is not None and not batched:
            raise ValueError("n_atoms goes with batches: types of shape (batch, atoms)")
        return Coords2GridFunction.apply(self.gmaker, self.center, coords, types, radii, *(() if n_atoms is None else (n_atoms,)))

    def extra_repr(self):
        return "resolution {:.2f}, dimension {}, center {:.3f},{:.3f},{:.3f}".format(
            self.gmaker.get_resolution(), self.gmaker.get_dimension(), *[float(c) for c in self.center])
