"""The operators on learned type vectors in 64 bits, written from their definitions, and how far a result held in 32 bits
and rounded once may be from them."""
import numpy as np
import torch

U = 2.0 ** -24                                # half a step of float32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(want, dtype):
    """Half a step of ``dtype`` at each value, that of the smallest normal number below it."""
    return want.abs().clamp(min=torch.finfo(dtype).tiny) * half_step(dtype) * (1 + 1e-6)


def philox(c, k):
    """One block of Philox4x32-10 on whole numbers."""
    c, k = list(c), list(k)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xffffffff, (a >> 32) ^ c[3] ^ k[1], a & 0xffffffff]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c


def draws(rows, width, rng, first=0):
    """(rows, width) draws of 32 bits as float64, of rows ``first`` and on."""
    seed, offset = rng
    groups = -(-width // 8)
    low = np.uint64(0xffffffff)
    halves = []
    for top in (0, 1 << 31):
        c = [np.broadcast_to(x, (rows, groups)).astype(np.uint64) for x in
             (np.arange(groups), np.arange(first, first + rows)[:, None], offset & 0xffffffff, offset >> 32 | top)]
        k = [np.uint64(seed & 0xffffffff), np.uint64(seed >> 32)]
        for _ in range(10):
            a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
            c = [(b >> np.uint64(32)) ^ c[1] ^ k[0], b & low, (a >> np.uint64(32)) ^ c[3] ^ k[1], a & low]
            k = [k[0] + np.uint64(0x9E3779B9) & low, k[1] + np.uint64(0xBB67AE85) & low]
        words = np.stack(c, -1).astype(np.float64)
        upper = np.floor(words / 65536.0)
        halves.append(np.stack([words - upper * 65536.0, upper], -1).reshape(rows, groups * 8)[:, :width])
    return halves[0] * 65536.0 + halves[1]


def factors(rows, width, p, rng, device="cuda"):
    """What dropout multiplies each value by, in 64 bits."""
    if p == 0:
        return torch.ones(rows, width, dtype=torch.float64, device=device)
    keep = draws(rows, width, rng) >= round(p * 2.0 ** 32)
    return torch.from_numpy(np.where(keep, 1.0 / (1.0 - p) if p < 1 else 0.0, 0.0)).to(device)


def filled(lead, n_atoms, device="cuda"):
    if n_atoms is None:
        return torch.ones(lead, dtype=torch.bool, device=device)
    return torch.arange(lead[1], device=device) < n_atoms.to(device)[:, None]


def valid_types(types, ntypes, n_atoms):
    """Rounded types, -1 where a slot is empty."""
    t = types.double() if types.is_floating_point() else types
    if types.is_floating_point():
        t = torch.where(t.isnan(), torch.full_like(t, -1.0), torch.sign(t) * torch.floor(t.abs() + 0.5)).clamp(-1, 2 ** 40)
    t = t.long()
    ok = (t >= 0) & (t < ntypes) & filled(types.shape, n_atoms, types.device)
    return torch.where(ok, t, torch.full_like(t, -1))


def embed(types, table, scale, n_atoms, p, rng):
    """(vectors, allowance before the last rounding): the product with the scale, the scale itself, the product with
    dropout's factor and that factor are rounded to float32."""
    V, W = table.shape
    t = valid_types(types, V, n_atoms).reshape(-1)
    rows = torch.cat([table.double(), torch.zeros(1, W, dtype=torch.float64, device=table.device)])[t]
    out = rows * scale * factors(t.numel(), W, p, rng)
    return out.view(tuple(types.shape) + (W,)), 4.1 * U * out.abs().view(tuple(types.shape) + (W,))


def embed_backward(types, diff, ntypes, scale, n_atoms, p, rng):
    """(table gradients, allowance): n terms, each rounded twice at most, summed in any order in float32, and the scale."""
    W = diff.shape[-1]
    t = valid_types(types, ntypes, n_atoms).reshape(-1)
    ok = t >= 0
    f = factors(t.numel(), W, p, rng)
    d = torch.where(ok[:, None] & (f != 0), diff.reshape(-1, W).double(), torch.zeros((), dtype=torch.float64, device=diff.device)) * f
    out, size, n = (torch.zeros(ntypes, k, dtype=torch.float64, device=diff.device) for k in (W, W, 1))
    out.index_add_(0, t[ok], d[ok])
    size.index_add_(0, t[ok], d[ok].abs())
    n.index_add_(0, t[ok], torch.ones(int(ok.sum()), 1, dtype=torch.float64, device=diff.device))
    return out * scale, (n + 4) * U * size * abs(scale)


def chain(width):
    """The longest chain of additions in a row's sum: a thread's own values, then the threads by pairs."""
    return max(32, -(-width // 32)) + 12


class Norm(object):
    """Layer norm of x in 64 bits with its allowances; errors as first-order bounds with a tenth to spare."""

    def __init__(self, x, weight, bias, eps, n_atoms):
        d64 = dict(dtype=torch.float64, device=x.device)
        self.on = filled(tuple(x.shape[:-1]), n_atoms, x.device)[..., None] if n_atoms is not None else \
            torch.ones(tuple(x.shape[:-1]) + (1,), dtype=torch.bool, device=x.device)
        W = self.width = x.shape[-1]
        self.x = torch.where(self.on, x.double(), torch.zeros((), **d64))
        self.w = torch.ones(W, **d64) if weight is None else weight.double()
        self.b = torch.zeros(W, **d64) if bias is None else bias.double()
        self.mean = self.x.mean(-1, keepdim=True)
        d = self.x - self.mean
        var = (d * d).mean(-1, keepdim=True)
        self.q = 1 / (var + eps).sqrt()
        self.h = d * self.q
        c = chain(W)
        dmean = (c + 2) * U * self.x.abs().mean(-1, keepdim=True)
        dd = dmean + U * d.abs()                                     # of x - mean
        self.dq = (dd.amax(-1, keepdim=True) * self.q + (c + 8) / 2 * U + 3 * U)   # of q, relative
        self.dmean = dmean
        self.dh = 1.1 * (self.q * dd + self.h.abs() * (self.dq + 2 * U))

    def forward(self):
        y = self.h * self.w + self.b
        tol = 1.1 * (self.w.abs() * (self.dh + 2 * U * self.h.abs()) + 2 * U * y.abs() + U * self.b.abs())
        zero = torch.zeros((), dtype=torch.float64, device=y.device)
        return torch.where(self.on, y, zero), torch.where(self.on, tol, zero)

    def backward(self, diff):
        """((dx, dw, db), their allowances); the sums over rows in any order."""
        zero = torch.zeros((), dtype=torch.float64, device=diff.device)
        g = torch.where(self.on, diff.double(), zero)
        a, h, q, c = g * self.w, self.h, self.q, chain(self.width)
        s0, s1 = a.mean(-1, keepdim=True), (a * h).mean(-1, keepdim=True)
        dx = q * (a - s0 - h * s1)
        e0 = (c + 4) * U * a.abs().mean(-1, keepdim=True)
        e1 = (a.abs() * self.dh).mean(-1, keepdim=True) + (c + 6) * U * (a * h).abs().mean(-1, keepdim=True)
        inner = a.abs() + s0.abs() + (h * s1).abs()
        tx = 1.1 * (q * (e0 + h.abs() * e1 + s1.abs() * self.dh + 5 * U * inner) + dx.abs() * self.dq)
        lead = tuple(range(g.dim() - 1))
        n = int(self.on.sum())
        dw, db = (g * h).sum(lead), g.sum(lead)
        tw = 1.1 * ((g.abs() * self.dh).sum(lead) + (n + 4) * U * (g * h).abs().sum(lead))
        tb = 1.1 * (n + 2) * U * g.abs().sum(lead)
        return (torch.where(self.on, dx, zero), dw, db), (torch.where(self.on, tx, zero), tw, tb)


def assert_near(got, want, tol):
    """``got`` within its own rounding and ``tol`` of ``want``, value by value."""
    allowed = tol + rounding(want, got.dtype)
    off = (got.double() - want).abs()
    bad = ~(off <= allowed)
    assert not bool(bad.any()), "%d of %d values off, worst %.3g of what is allowed at %s" % (
        int(bad.sum()), bad.numel(), float((off / allowed).nan_to_num(1e300).max()), tuple(bad.nonzero()[0].tolist()))
