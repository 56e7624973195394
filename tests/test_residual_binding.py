"""What the binding of the residual stream's operators does with its arguments before the library sees them.  Host tensors
stand for a device's: the entry points of the library are replaced, so nothing here reaches a kernel."""
import ctypes as C

import pytest
import torch

from flagcx_amd import local as L

INV = int(L.Result.InvalidArgument)


class Entry:
    """Stands for the library: notes the arguments of the calls that would run, hands the rest through."""

    def __init__(self, real):
        self.real, self.calls = real, []

    def __getattr__(self, name):
        if name.endswith("Workspace") or name in ("flagcxLocalGetErrorString", "flagcxLocalGetLastError"):
            return getattr(self.real, name)

        def note(*args):
            for cast, a in zip(getattr(self.real, name).argtypes, args):
                if cast in (C.c_size_t, C.c_int64, C.c_int):
                    assert cast(a).value == a, (name, a)  # what the library would be handed is what was asked for
            self.calls.append((name, args))
            return 0
        return note


@pytest.fixture()
def entry(monkeypatch):
    e = Entry(L.lib())
    monkeypatch.setattr(L, "lib", lambda: e)
    monkeypatch.setattr(L, "_device", lambda t: -1)  # where host tensors are
    monkeypatch.setattr(L, "_stream_ref", lambda stream, device: None)
    monkeypatch.setattr(L, "_workspace", lambda ws, need, device, stream: (1 << 20, need, None))
    return e


def refused(call):
    with pytest.raises(L.FlagcxError) as e:
        call()
    assert e.value.code == INV
    return str(e.value)


@pytest.mark.parametrize("gate_rows", [-1, 1 << 64, (1 << 64) + 2, (1 << 65) + 4])
def test_gate_rows_beyond_64_bits_are_refused(entry, gate_rows):
    """2^64 + 2 would be cut to groups of two rows, of which the one row of gates here holds the first."""
    x, gate = torch.zeros(10, 8), torch.zeros(1, 8)
    out, y = torch.zeros_like(x), torch.zeros_like(x)
    assert "gate_rows" in refused(lambda: L.reduce_norm([x], x, out, y, gate=gate, gate_rows=gate_rows))
    assert "gate_rows" in refused(lambda: L.reduce_norm_backward(x, x, x, out, total=x, gate=gate, gate_rows=gate_rows))
    assert "gate_rows" in refused(lambda: L.reduce_norm_backward(x, x, x, out, total=x, gate=gate, gate_rows=gate_rows,
                                                                 gate_grad=torch.zeros_like(gate)))
    assert not entry.calls
    for n in (0, 10, 11, (1 << 64) - 1):
        L.reduce_norm([x], x, out, y, gate=gate, gate_rows=n)
        assert entry.calls.pop()[1][0].gaterows == n


@pytest.mark.parametrize("first", [1 << 63, -(1 << 63) - 1, 1 << 64, (1 << 64) + 3, -(1 << 64)])
def test_first_beyond_64_bits_is_refused(entry, first):
    table, ids, out = torch.zeros(6, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(4, 8)
    assert "first" in refused(lambda: L.embedding(table, ids, out, first=first))
    assert "first" in refused(lambda: L.embedding_grad(out, ids, table, first=first))
    assert not entry.calls
    for n in (0, 5, -7, (1 << 63) - 1, -(1 << 63)):
        L.embedding(table, ids, out, first=n)
        L.embedding_grad(out, ids, table, first=n)
    assert len(entry.calls) == 10


def test_workspaces_of_sizes_beyond_64_bits_are_refused():
    for big in (-1, 1 << 64, (1 << 64) + 4):
        assert "rows" in refused(lambda: L.reduce_norm_backward_workspace(big, 64))
        assert "dim" in refused(lambda: L.reduce_norm_backward_workspace(4, big))
        assert "gate_rows" in refused(lambda: L.reduce_norm_backward_workspace(4, 64, True, big))
        assert "tokens" in refused(lambda: L.embedding_grad_workspace(big, 10, 64))
        assert "vocab" in refused(lambda: L.embedding_grad_workspace(600, big, 64))
        assert "dim" in refused(lambda: L.embedding_grad_workspace(600, 10, big))


def test_weight_gradient_without_a_gradient_of_the_norm(entry):
    """norm_grad=None stands for zeros: the weight's gradient is then zeros, which the entry point writes."""
    x, w = torch.zeros(10, 8), torch.ones(8)
    out, dw = torch.zeros_like(x), torch.zeros_like(w)
    L.reduce_norm_backward(x, None, x, out, total=x, pre_weight=w, pre_weight_grad=dw)
    name, args = entry.calls.pop()
    end = args[0]
    assert name == "flagcxLocalReduceNormBackward" and end.norms == L.NORM_PRE and end.preweight == w.data_ptr()
    assert args[3] == x.data_ptr() and args[5] is None and args[14] == dw.data_ptr()
    L.reduce_norm_backward(x, None, x, out, total=x, pre_weight=w)  # no part of that norm is asked for
    assert entry.calls.pop()[1][0].norms == 0
