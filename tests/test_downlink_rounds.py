"""CPU test of the way down over rounds: a client that missed a vector, or is
given one twice, is told so (the kernels' calls replaced by plain sums); the
round's number reaches other ranks with the vector."""
import os
import socket

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def plain(monkeypatch):
    """encode and decode in float32: the codes of element i are its change, kept aside."""
    from compressor_b200 import mx4
    changes = {}

    def encode(x, base=None, rounding="nearest", seed=0, counter=None):
        sent = mx4.Mx4Vector.empty(x.numel(), "cpu")
        changes[id(sent)] = (sent, x.float() - base)
        base += changes[id(sent)][1]
        return sent

    def decode(sent, out=None, weight=1.0, accumulate=False, dtype=torch.float32):
        out += changes[id(sent)][1]
        return out

    monkeypatch.setattr(mx4, "_check", lambda t, what: None)
    monkeypatch.setattr(mx4, "encode", encode)
    monkeypatch.setattr(mx4, "decode", decode)


def test_who_missed_a_round_is_told(plain):
    from compressor_b200 import federated as fed
    from compressor_b200.mx4 import Mx4Vector
    weights = torch.zeros(40)
    down = fed.Downlink(weights)
    mine, sents = weights.clone(), []
    for t in range(4):
        weights += t + 1
        sents.append(down.send())
    assert [int(s.round) for s in sents] == [0, 1, 2, 3] and int(down.round) == 4
    assert fed.Downlink.receive(sents[0], mine, round=0) is mine
    for wrong, at in ((sents[0], 1), (sents[2], 1), (Mx4Vector.empty(40, "cpu"), 1)):   # twice; one too far; of no round
        with pytest.raises(ValueError, match="round"):
            fed.Downlink.receive(wrong, mine, round=at)
    assert (mine == 1).all()
    for t in (1, 2, 3):
        fed.Downlink.receive(sents[t], mine, round=t)
    assert torch.equal(mine, weights) and torch.equal(down.held, weights)
    fed.Downlink.receive(sents[3], mine)   # unasked nothing is checked
    # after a restart the numbers go on
    again = fed.Downlink(weights, held=down.held)
    again.round.copy_(down.round)
    assert int(again.send().round) == 4


def _rank(rank, world, port, path):
    import torch.distributed as dist
    from compressor_b200 import federated as fed
    from compressor_b200.mx4 import Mx4Vector
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        got = []
        sent = Mx4Vector.empty(33, "cpu")
        for t in (7, None, 9):   # (a receiver uses its vector again)
            if rank == 0:
                sent.round = None if t is None else torch.tensor([t])
                sent.buffer.fill_(t or 1)
            fed.broadcast(sent, dist)
            got += [int(sent.round), int(sent.buffer[0])]
        torch.save(got, f"{path}/{rank}.pt")
    finally:
        dist.destroy_process_group()


def test_the_number_goes_with_the_vector(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    torch.multiprocessing.spawn(_rank, args=(2, port, str(tmp_path)), nprocs=2)
    for r in range(2):
        assert torch.load(tmp_path / f"{r}.pt") == [7, 7, -1, 1, 9, 9]
