"""CPU test of the way down over several ranks: the bytes of a 4-bit vector and
of a matrix reach every rank whole (federated.broadcast, two gloo ranks)."""
import os
import socket

import pytest

torch = pytest.importorskip("torch")


def _rank(rank, world, port, path):
    import torch.distributed as dist
    from compressor_b200 import federated as fed
    from compressor_b200.mx4 import Mx4Matrix, Mx4Vector
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        got = []
        for i, n in enumerate((1, 33, 5130)):
            sent = Mx4Vector.empty(n, "cpu")
            if rank == 1:
                sent.buffer.copy_(torch.arange(sent.buffer.numel()) * (7 + i) % 251)
            fed.broadcast(sent, dist, src=1)
            got += [sent.codes.clone(), sent.scales.clone()]
        m = Mx4Matrix.empty(9, 300, "cpu")
        m.buffer.fill_(0 if rank else 5)
        fed.broadcast(m, dist)
        torch.save(got + [m.buffer], f"{path}/{rank}.pt")
    finally:
        dist.destroy_process_group()


def test_broadcast_reaches_every_rank(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    torch.multiprocessing.spawn(_rank, args=(2, port, str(tmp_path)), nprocs=2)
    a, b = (torch.load(tmp_path / f"{r}.pt") for r in range(2))
    assert len(a) == 7 and all(torch.equal(x, y) for x, y in zip(a, b))
    assert [x.numel() for x in a[:6]] == [1, 1, 17, 2, 2565, 161] and (a[6] == 5).all()
    assert torch.equal(a[4], (torch.arange(2565) * 9 % 251).to(torch.uint8))


def test_broadcast_on_one_rank_changes_nothing():
    from compressor_b200 import federated as fed
    from compressor_b200.mx4 import Mx4Vector
    v = Mx4Vector.empty(40, "cpu")
    v.buffer.fill_(3)
    fed.broadcast(v, None)
    assert (v.buffer == 3).all()
