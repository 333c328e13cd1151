"""The operators on learned type vectors, one pass each: what a network does with atom types before they are gridded.

A case is a dict of plain values; ``op`` says which operator it calls:

* ``embed``: type indices to rows of a table (``embed_types``), with ``train`` the table's gradient too.
* ``norm``: layer norm over the last dimension, with ``train`` the gradients of inputs, weights and biases too.
* ``dropout``: values dropped by a counter-based generator; the gradient is the same call on the gradient.
* ``vectors``: all of them as a network uses them in a training step - the table normalised, looked up and dropped,
  then the gradients back to the table, the weights and the biases.

``batch`` 0 is one example without counts, a positive one a padded batch of ``min_atoms`` to ``atoms`` atoms an
example.  Types follow a Zipf distribution, as those of atoms and fragments do, and one in fifty is -1 (an atom that
the typer does not map).  ``dtype`` is that of vectors and their gradients, ``table`` that of the table (in ``vectors``
float32, as a network's parameters are) and ``weights`` that of a layer norm's parameters; ``index`` is that of the type
indices (float32 is what the example provider hands out).

Draws of the generator: 32 bits for each value, Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers:
as easy as 1, 2, 3", 2011) under the key ``seed``.  A block's counter is (column / 8, row, offset as two words); value j of
its eight columns takes the j-th half word as its upper bits, and as its lower bits that of the block with the
counter's topmost bit set.  It is dropped where the draw is below p * 2^32.
"""
import math

import numpy as np
import torch

own = False
EPS = 1e-5
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16,
          "int32": torch.int32, "int64": torch.int64}


def listed():
    embed = dict(op="embed", train=True, batch=50, min_atoms=2000, atoms=4000, types=28, width=28, dtype="float32",
                 table="float32", index="float32", scale=1.0, p=0.0)
    norm = dict(op="norm", train=True, batch=50, min_atoms=2000, atoms=4000, width=28, dtype="float32",
                weights="float32")
    drop = dict(op="dropout", batch=0, atoms=40, width=32, dtype="float32", p=0.1)
    return [
        # one ligand's atoms to vectors: scoring a pose at a time, nothing but latency
        dict(embed, name="ligand types", train=False, batch=0, atoms=40, types=14, width=32),
        # the training batch of a docking network that learns its types: every table row is hit by thousands of atoms
        dict(embed, name="learned types"),
        # fragments as types: a large table of wide rows, most of them not met in a step
        dict(embed, name="fragment types", batch=0, atoms=16384, types=50021, width=1024, dtype="bfloat16",
             table="bfloat16", index="int64", scale=32.0),
        # ligands beside pockets, rows of no convenient alignment, dropped as they are looked up
        dict(embed, name="odd types", batch=17, min_atoms=37, atoms=1503, types=350, width=45, dtype="float16",
             index="int32", scale=0.5, p=0.25),
        # one ligand's vectors normalised
        dict(norm, name="ligand norm", train=False, batch=0, atoms=40, width=32),
        # the vectors of the training batch
        dict(norm, name="norm of atoms"),
        # the wide features of a large network
        dict(norm, name="wide norm", batch=0, atoms=16384, width=4096, dtype="bfloat16", weights="float32"),
        # features of no convenient width
        dict(norm, name="odd norm", batch=17, min_atoms=37, atoms=1503, width=1001, dtype="float16", weights="float16"),
        # one ligand's vectors dropped
        dict(drop, name="ligand dropout"),
        # wide features of a large network
        dict(drop, name="wide dropout", atoms=8192, width=4096, dtype="bfloat16", p=0.5),
        # features of no convenient width
        dict(drop, name="odd dropout", batch=17, min_atoms=37, atoms=1503, width=333, p=0.2),
        # a training step of the input vectors
        dict(op="vectors", name="type vectors", batch=50, min_atoms=2000, atoms=4000, types=28, width=32, dtype="float32",
             weights="float32", index="float32", p=0.1),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed", "norm", "norm", "dropout", "vectors"])
    batch = rng.choice([0, _spread(rng, 2, 64)])
    atoms = _spread(rng, 1, 65536) if batch == 0 else _spread(rng, 16, 4000)
    rows = max(1, batch) * atoms
    # the layer norm of a few values is next to nothing but its rounding
    width = min(_spread(rng, 8 if op in ("norm", "vectors") else 1, 8192), (1 << 25) // rows)
    if rng.random() < 0.5:
        width = max(1, width // 8 * 8)
    case = dict(op=op, batch=batch, atoms=atoms, width=width, dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]))
    if batch:
        case["min_atoms"] = max(1, int(atoms * rng.uniform(0.02, 1.0)))
    if op in ("embed", "vectors"):
        case.update(types=min(_spread(rng, 2, 100000), (1 << 25) // width), index=rng.choice(["float32", "int32", "int64"]))
        if op == "vectors":
            case["types"] = min(case["types"], max(2, rows), (1 << 23) // width)
    if op in ("embed", "norm"):
        case["train"] = rng.random() < 0.7
    if op == "embed":
        case.update(scale=round(rng.uniform(0.1, 40.0), 3), p=rng.choice([0.0, 0.0, 0.1, 0.3]),
                    table=rng.choice(["float32", case["dtype"]]))
    if op in ("norm", "vectors"):
        case["weights"] = rng.choice(["float32", case["dtype"]]) if op == "norm" else "float32"
    if op in ("dropout", "vectors"):
        case["p"] = round(rng.uniform(0.01, 0.7), 4)
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, B, N, W = case["op"], case["batch"], case["atoms"], case["width"]
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    lead = (B, N) if B else (N,)
    s = dict(case=case, p=case.get("p", 0.0), scale=case.get("scale", 1.0), n_atoms=None, train=case.get("train", True))
    words = torch.randint(0, 1 << 31, (2,), generator=g, device="cuda").tolist()
    s["rng"] = (words[0] << 31 | words[1], words[1])
    if B and op != "dropout":
        s["n_atoms"] = torch.randint(case["min_atoms"], N + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    if op in ("embed", "vectors"):
        V = case["types"]
        order = torch.randperm(V, generator=g, device="cuda")
        u = torch.rand(lead, generator=g, device="cuda", dtype=torch.float64)
        rank = (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp(0, V - 1)
        types = order[rank]
        types[torch.rand(lead, generator=g, device="cuda") < 0.02] = -1
        s["types"] = types.to(DTYPES[case["index"]])
        s["table"] = normal(V, W).to(DTYPES[case.get("table", "float32")])
        s["out"] = torch.empty(lead + (W,), dtype=dtype, device="cuda")
        s["table_gradients"] = torch.empty_like(s["table"])
    else:
        s["x"] = (normal(*lead, W) * (0.5 + torch.rand(lead + (1,), generator=g, device="cuda")) + normal(*lead, 1)).to(dtype)
        s["out"] = torch.empty_like(s["x"])
    if op in ("norm", "vectors"):
        wtype = DTYPES[case["weights"]]
        s["weight"] = (1.0 + 0.2 * normal(W)).to(wtype)
        s["bias"] = (0.2 * normal(W)).to(wtype)
        rows = s["table"] if op == "vectors" else s["x"]
        s["stats"] = torch.empty(rows.shape[:-1] + (2,), device="cuda")
        s["normed"] = torch.empty_like(rows)
        s["row_gradients"] = torch.empty_like(rows)
        s["weight_gradients"], s["bias_gradients"] = torch.empty_like(s["weight"]), torch.empty_like(s["bias"])
    if op != "dropout":
        s["diff"] = normal(*lead, W).to(dtype)
    return s


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    import libmolgrid_b200 as lmg
    op, p, na = s["case"]["op"], s["p"], s["n_atoms"]
    rng = s["rng"] if p else None
    if op == "embed":
        lmg.embed_types(s["types"], s["table"], s["out"], s["scale"], na, p, rng)
        if not s["train"]:
            return {"out": s["out"]}
        lmg.embed_types_backward(s["types"], s["diff"], s["table_gradients"], s["scale"], na, p, rng)
        return {"out": s["out"], "table": s["table_gradients"]}
    if op == "norm":
        lmg.layer_norm(s["x"], s["weight"], s["bias"], s["normed"], s["stats"], EPS, na)
        if not s["train"]:
            return {"out": s["normed"]}
        lmg.layer_norm_backward(s["x"], s["weight"], s["stats"], s["diff"], s["row_gradients"], s["weight_gradients"],
                                s["bias_gradients"], na)
        return {"out": s["normed"], "x": s["row_gradients"], "weight": s["weight_gradients"], "bias": s["bias_gradients"]}
    if op == "dropout":
        lmg.dropout(s["x"], s["out"], p, rng)
        return {"out": s["out"]}
    lmg.layer_norm(s["table"], s["weight"], s["bias"], s["normed"], s["stats"], EPS)
    lmg.embed_types(s["types"], s["normed"], s["out"], 1.0, na, p, rng)
    lmg.embed_types_backward(s["types"], s["diff"], s["table_gradients"], 1.0, na, p, rng)
    lmg.layer_norm_backward(s["table"], s["weight"], s["stats"], s["table_gradients"], s["row_gradients"],
                            s["weight_gradients"], s["bias_gradients"])
    return {"out": s["out"], "table": s["row_gradients"], "weight": s["weight_gradients"], "bias": s["bias_gradients"]}


# ---- the plain form ---------------------------------------------------------------------------------------------------
def _kept(rows, width, p, rng):
    """(rows, width): which values stay."""
    seed, offset = rng
    low, groups = 0xffffffff, -(-width // 8)

    def pair(a, b):
        return torch.tensor([a, b], device="cuda").view(2, 1, 1, 1)

    # words 0 and 2 of each counter in x, 1 and 3 in y, 32 bits held in 64; (pair, with the topmost bit or without, row, group)
    x, y = (torch.empty((2, 2, rows, groups), dtype=torch.int64, device="cuda") for _ in range(2))
    x[0], x[1] = torch.arange(groups, device="cuda"), offset & low
    y[0], y[1] = torch.arange(rows, device="cuda")[:, None], offset >> 32
    y[1, 1] |= 1 << 31
    factor, step = pair(0xD2511F53, 0xCD9E8D57), pair(0x9E3779B9, 0xBB67AE85)
    key = pair(seed & low, seed >> 32 & low)
    for _ in range(10):
        product = (x * factor).flip(0)
        x, y = (product >> 32 & low) ^ y ^ key, product & low
        key = key + step & low
    words = torch.stack([x[0], y[0], x[1], y[1]], -1)
    upper, lower = torch.stack([words & 0xffff, words >> 16], -1).reshape(2, rows, groups * 8)[..., :width]
    return (upper << 16 | lower) >= int(round(p * 2.0 ** 32))


def _dropped(x, p, rng):
    """x (float32) after dropout over its last dimension."""
    if not p:
        return x
    kept = _kept(x.numel() // x.shape[-1], x.shape[-1], p, rng).view(x.shape)
    return torch.where(kept, x * (1.0 / (1.0 - p)), torch.zeros((), device="cuda"))


def _filled(lead, n_atoms):
    """Which slots of a padded batch hold atoms."""
    if n_atoms is None:
        return torch.ones(lead, dtype=torch.bool, device="cuda")
    return torch.arange(lead[1], device="cuda") < n_atoms[:, None]


def _normalised(x, s, n_atoms):
    """(out, h, 1 / deviation, filled) of layer norm in 32 bits."""
    filled = _filled(x.shape[:-1], n_atoms)[..., None]
    x = x.float()
    d = x - x.mean(-1, keepdim=True)
    q = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
    h = d * q
    out = torch.where(filled, h * s["weight"].float() + s["bias"].float(), torch.zeros((), device="cuda"))
    return out, h, q, filled


def _norm_gradients(g, h, q, filled, s):
    g = torch.where(filled, g.float(), torch.zeros((), device="cuda"))
    a = g * s["weight"].float()
    dx = q * (a - a.mean(-1, keepdim=True) - h * (a * h).mean(-1, keepdim=True))
    lead = tuple(range(g.dim() - 1))
    return dx, (g * h).sum(lead), g.sum(lead)


def _plain(s):
    op, p, rng = s["case"]["op"], s["p"], s["rng"]
    dtype = DTYPES[s["case"]["dtype"]]
    if op == "dropout":
        return {"out": _dropped(s["x"].float(), p, rng).to(dtype)}
    if op == "norm":
        out, h, q, filled = _normalised(s["x"], s, s["n_atoms"])
        if not s["train"]:
            return {"out": out.to(dtype)}
        dx, dw, db = _norm_gradients(s["diff"], h, q, filled, s)
        return {"out": out.to(dtype), "x": dx.to(dtype), "weight": dw.to(s["weight"].dtype), "bias": db.to(s["weight"].dtype)}
    types, V = s["types"].long(), s["table"].shape[0]
    there = (types >= 0) & _filled(types.shape, s["n_atoms"])
    table = s["table"]
    if op == "vectors":
        table, h, q, filled = _normalised(s["table"], s, None)
    rows = table.float()[types.clamp(min=0).masked_fill(~there, 0)] * s["scale"]
    out = _dropped(torch.where(there[..., None], rows, torch.zeros((), device="cuda")), p, rng).to(dtype)
    if not s["train"]:
        return {"out": out}
    grad = _dropped(s["diff"].float(), p, rng) * s["scale"]
    dtable = torch.zeros(table.shape, device="cuda").index_add_(0, types[there], grad[there])
    if op == "embed":
        return {"out": out, "table": dtable.to(s["table"].dtype)}
    dx, dw, db = _norm_gradients(dtable, h, q, filled, s)
    return {"out": out, "table": dx, "weight": dw.to(s["weight"].dtype), "bias": db.to(s["weight"].dtype)}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def _factors(rows, width, p, rng):
    """What dropout multiplies each value by."""
    seed, offset = rng
    mask, shift = np.uint64(0xffffffff), np.uint64(32)
    draws = []
    for top in (0, 1 << 31):
        key = [np.uint64(seed & 0xffffffff), np.uint64(seed >> 32)]
        x0 = np.broadcast_to(np.arange(-(-width // 8), dtype=np.uint64), (rows, -(-width // 8)))
        x1 = np.broadcast_to(np.arange(rows, dtype=np.uint64)[:, None], x0.shape)
        x2, x3 = np.uint64(offset & 0xffffffff), np.uint64(offset >> 32 | top)
        for i in range(10):
            m0, m1 = np.uint64(0xD2511F53) * x0, np.uint64(0xCD9E8D57) * x2
            x0, x1, x2, x3 = (m1 >> shift) ^ x1 ^ key[0], m1 & mask, (m0 >> shift) ^ x3 ^ key[1], m0 & mask
            key = [key[0] + np.uint64(0x9E3779B9) & mask, key[1] + np.uint64(0xBB67AE85) & mask]
        halves = np.stack([x.astype(np.uint32) for x in (x0, x1, x2, x3)], -1).view(np.uint16)
        draws.append(halves.reshape(rows, -1)[:, :width].astype(np.float64))
    return np.where(draws[0] * 65536.0 + draws[1] < round(p * 2.0 ** 32), 0.0, 1.0 / (1.0 - p))


def _wide(t):
    return t.detach().double().cpu().numpy()


def _norm_exact(x, w, b, g, empty):
    """Layer norm and its gradients by differentiation, in 64 bits."""
    x, w, b = (t.detach().double().requires_grad_() for t in (x, w, b))
    v, m = torch.var_mean(x, -1, correction=0, keepdim=True)
    y = ((x - m) / (v + EPS).sqrt() * w + b).masked_fill(empty[..., None], 0.0)
    return (y.detach(),) + torch.autograd.grad(y, (x, w, b), g.double())


def exact(case, seed):
    s = prepare(case, seed)
    op, W, na = case["op"], case["width"], s["n_atoms"]
    if op == "dropout":
        x = _wide(s["x"])
        return {"out": x * _factors(x.size // W, W, s["p"], s["rng"]).reshape(x.shape)}
    lead = s["diff"].shape[:-1]
    empty = torch.zeros(lead, dtype=torch.bool, device="cuda")
    if na is not None:
        empty = torch.arange(lead[1], device="cuda").expand(lead) >= na[:, None]
    if op == "norm":
        out, dx, dw, db = _norm_exact(s["x"], s["weight"], s["bias"], s["diff"], empty)
        return {"out": out, "x": dx, "weight": dw, "bias": db} if s["train"] else {"out": out}
    types = np.where(empty.cpu().numpy(), -1, s["types"].cpu().numpy()).astype(np.int64).reshape(-1)
    V, R = case["types"], types.size
    none = torch.zeros(V, dtype=torch.bool, device="cuda")
    norm = (s["table"], s["weight"], s["bias"]) if op == "vectors" else None
    table = _wide(_norm_exact(*norm, torch.zeros_like(s["table"]), none)[0] if norm else s["table"])
    out = np.concatenate([table, np.zeros((1, W))])[types] * s["scale"]
    grad = _wide(s["diff"]).reshape(R, W) * s["scale"]
    if s["p"]:
        f = _factors(R, W, s["p"], s["rng"])
        out, grad = out * f, grad * f
    order = np.argsort(types, kind="stable")
    order = order[np.searchsorted(types[order], 0):]
    dtable = np.zeros((V, W))
    if order.size:
        met, first = np.unique(types[order], return_index=True)
        dtable[met] = np.add.reduceat(grad[order], first, axis=0)
    out = out.reshape(s["out"].shape)
    if op == "embed":
        return {"out": out, "table": dtable} if s["train"] else {"out": out}
    _, dx, dw, db = _norm_exact(*norm, torch.from_numpy(dtable).cuda(), none)
    return {"out": out, "table": dx, "weight": dw, "bias": db}


def work(case):
    op, W = case["op"], case["width"]
    R = max(1, case["batch"]) * case["atoms"]
    size = 4 if case["dtype"] == "float32" else 2
    wsize = 4 if case.get("weights") == "float32" else 2
    train = case.get("train", True)
    if op == "dropout":
        return {"bytes": 2 * R * W * size, "flops": R * W}
    if case["batch"]:   # slots that hold atoms, on average; the others are written only
        held = case["batch"] * (case["min_atoms"] + case["atoms"]) / 2
    else:
        held = R
    if op == "norm":
        return {"bytes": (R + held + (R + 2 * held if train else 0)) * W * size + (5 if train else 2) * W * wsize,
                "flops": held * W * (22 if train else 8)}
    index = {"int64": 8}.get(case["index"], 4) * held
    V = case["types"]
    tsize = 2 if case.get("table", "float32") != "float32" else 4
    out = {"bytes": index + min(V, held) * W * tsize + R * W * size, "flops": held * W}
    if train:
        out["bytes"] += held * W * size + V * W * tsize
        out["flops"] += 2 * held * W
    if op == "vectors":
        out["bytes"] += V * W * tsize + 5 * W * wsize
        out["flops"] += V * W * 22
    return out
