"""Learned type vectors without a GPU: what their calls plan and refuse at the ends of their ranges."""
import copy
import ctypes
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def test_rows_of_a_thread_begin_alike(lib):
    """A thread of a layer norm copies whole pieces of 16 bytes and keeps the place in them at which its first row begins: where rows do not
    begin on 16 bytes, what it jumps by has to be a multiple of the values that 16 bytes hold, or it has one row alone."""
    rows = list(range(1, 20)) + [31, 32, 33, 64, 127, 128, 129, 147, 148, 149, 295, 296, 297, 443, 444, 445, 591, 592, 593, 600, 888, 889, 1184,
                                 1185, 2367, 2368, 2400, 4736, 5000, 9471, 9472, 20000]
    plan = (ctypes.c_uint * 5)()
    broken = []
    for slack in (3, 7):
        for width in range(1, 8193):
            for n in rows:
                lib.lmg_norm_plan(n, width, slack, plan)
                wide, at_once, times, forward, backward = plan
                if wide:
                    continue
                assert times == -(-n // at_once) and 1 <= forward <= times and 1 <= backward <= times
                # the jump in values is at_once * blocks * ld, for any ld
                broken += [(slack, width, n, b) for b in (forward, backward) if b < times and at_once * b % (slack + 1)]
    assert not broken, (len(broken), broken[:5])


@pytest.mark.parametrize("slack", [0, 3, 7])
def test_workspace_covers_every_alignment(lib, slack):
    from libmolgrid_b200 import _cabi
    plan = (ctypes.c_uint * 5)()
    for width in (1, 28, 64, 505, 506, 1001, 4096, 8185, 8192, 9000):
        for n in (1, 2, 3, 4, 5, 100, 1000, 20000):
            lib.lmg_norm_plan(n, width, slack, plan)
            assert lib.lmg_vectors_workspace_bytes(_cabi.OP_LAYER_NORM_BACKWARD, n, 0, width) >= 256 + plan[4] * 2 * width * 4


def test_draws_go_with_type_indices():
    import libmolgrid_b200 as lmg
    with pytest.raises(ValueError):
        lmg.Coords2Grid(lmg.GridMaker(0.5, 5.5))(torch.zeros(2, 4, 3), torch.zeros(2, 4, 2), torch.ones(2, 4), draw=(1, 0))
    assert lmg.Dropout(0.0).draw() is None and lmg.TypeVectors(3, 2, p=0.5).eval().draw() is None


# ---- what is a rank's own ---------------------------------------------------------------------------------------------
def _rank(rank, port, out):
    import libmolgrid_b200 as lmg
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=2)

    class Network(torch.nn.Module):   # its pass is on the host: what is tested is what the wrapper copies between ranks before it
        def __init__(self):
            super().__init__()
            self.types, self.drop, self.rest = lmg.TypeVectors(5, 4, p=0.5, seed=100 + rank), lmg.Dropout(0.5, seed=200 + rank), torch.nn.Linear(4, 4)

        def forward(self, x):
            return self.rest(x) + self.types.table.sum() + self.types.weight.sum() + self.types.bias.sum()

    net = torch.nn.parallel.DistributedDataParallel(Network())
    mine = net.module
    mine.types.generator[1] = 7 + rank
    mine.types.status[0] = rank        # a type beyond the table, on one rank
    for _ in range(2):
        net(torch.ones(2, 4)).sum().backward()
    out.put((rank, mine.types.generator.tolist(), mine.drop.generator.tolist(), int(mine.types.status), float(mine.types.table.detach().sum())))
    dist.barrier()
    dist.destroy_process_group()


def test_ranks_keep_their_generators_and_status():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    out = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, port, out)) for r in range(2)]
    for p in procs:
        p.start()
    got = sorted(out.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(timeout=120)
    assert [g[1:4] for g in got] == [([100, 7], [200, 0], 0), ([101, 8], [201, 0], 1)]
    assert got[0][4] == got[1][4]      # parameters are the ranks' common ones


def test_generators_in_state_dicts():
    import libmolgrid_b200 as lmg
    m = torch.nn.Sequential(lmg.TypeVectors(5, 4, p=0.5, seed=3), lmg.Dropout(0.5, seed=4))
    m[0].generator[1] = 11
    state = m.state_dict()
    assert set(state) == {"0.table", "0.weight", "0.bias", "0.generator", "1.generator"}
    for assign in (False, True):
        twin = torch.nn.Sequential(lmg.TypeVectors(5, 4, p=0.5), lmg.Dropout(0.5))
        assert not any(twin.load_state_dict({k: v.clone() for k, v in state.items()}, assign=assign))
        assert twin[0].generator.tolist() == [3, 11] and twin[1].generator.tolist() == [4, 0]
    twin = copy.deepcopy(m)
    twin[0].generator[1] = 12
    assert m[0].generator.tolist() == [3, 11] and twin[0].generator.tolist() == [3, 12]
    del state["1.generator"]
    with pytest.raises(RuntimeError, match="Missing"):
        twin.load_state_dict(state)
    assert twin.load_state_dict(state, strict=False).missing_keys == ["1.generator"]
    with pytest.raises(RuntimeError, match="generator"):
        twin.load_state_dict(dict(state, **{"1.generator": torch.zeros(3)}))
    m = m.half().to("meta")
    assert m[0].generator.dtype is torch.int64 and m[0].generator.is_meta and m[0].status.is_meta and m[0].table.dtype is torch.float16


@pytest.mark.parametrize("bad", [dict(scale=1e20), dict(scale=1e-25), dict(scale=1e200), dict(scale=1e-200), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(eps=0.0), dict(eps=-1e-5), dict(eps=1e-44), dict(eps=float("nan"))])
def test_scales_that_take_eps_out_of_range(bad):
    """The norm of scale * row is that of the row with eps / scale^2, which float32 has to hold."""
    import libmolgrid_b200 as lmg
    with pytest.raises(ValueError):
        lmg.TypeVectors(3, 2, **bad)
    lmg.TypeVectors(3, 2, scale=1e16)
    lmg.TypeVectors(3, 2, scale=1e-21)
    if "scale" in bad:
        lmg.TypeVectors(3, 2, norm=False, **bad)
