"""Dropout's call of the library on the CPU, the library being a stand-in: what
a call points to is alive while the call is made."""
import weakref

import pytest

torch = pytest.importorskip("torch")

from compressor_b200 import dropout, mx4  # noqa: E402

copies = []


class Watched(torch.Tensor):
    """A tensor that remembers, weakly, the copies that contiguous() made of it."""

    def contiguous(self, *args, **kwargs):
        c = self.as_subclass(torch.Tensor).contiguous(*args, **kwargs)
        copies.append((c.data_ptr(), weakref.ref(c)))
        return c


class Library:
    """Takes falcom_dropout's place; keeps its arguments and which copies were alive."""

    def falcom_dropout(self, x, residual, y, dtype, rows, cols, args, stream):
        self.args, self.alive = (x, residual, rows, cols), [(at, ref() is not None) for at, ref in copies]
        return 0


@pytest.mark.parametrize("strided", ["x", "residual", "both"])
def test_copies_live_while_the_call_is_made(monkeypatch, strided):
    lib = Library()
    monkeypatch.setattr(mx4, "_library", lambda: lib)
    monkeypatch.setattr(mx4, "_stream", lambda device: None)
    copies.clear()
    x, r = torch.randn(6, 4), torch.randn(6, 4)
    if strided != "residual":
        x = torch.randn(4, 6).t().as_subclass(Watched)
    if strided != "x":
        r = torch.randn(4, 6).t().as_subclass(Watched)
    y = dropout._run(x, r, 0.5, 1, None)
    assert y.shape == (6, 4) and len(copies) == (2 if strided == "both" else 1)
    assert lib.args[2:] == (6, 4) and [a for a, _ in lib.alive] == [a for a, t in zip(lib.args, (x, r)) if isinstance(t, Watched)]
    assert all(alive for _, alive in lib.alive)
