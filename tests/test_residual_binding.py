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


def table_plan(tokens, vocab, dim):
    """What a table gradient of these sizes writes to its workspace: sorted tokens, digit counts, flags, partial rows."""
    up = lambda a, b: -(-a // b)
    bits = max(1, vocab.bit_length())
    bits = up(bits, up(bits, 11))
    per = up(up(tokens, min(up(tokens, 2048), 256)), 512) * 512
    chunk = 8
    while chunk < 32 and tokens * up(dim, 512) // chunk > 4096:
        chunk *= 2
    return 16 * tokens + up(tokens, per) * (4 << bits) + vocab + up(tokens, chunk) * 2 * up(dim, 4) * 4 * 4


def test_table_workspace_of_the_largest_call_serves_smaller_ones():
    """The size holds what a call writes and does not fall as tokens, vocab or dim grow."""
    tokens = [1, 255, 256, 257, 300, 2047, 2048, 2049, 4096, 4097, 8191, 8192, 16384, 16393, 32768, 32769, 32777, 32784, 40000,
              65543, 65551, 65552, 131072, 131080, 262144, 524288, 524289, 530000, 1 << 20, (1 << 20) + 1, (1 << 31) - 1]
    vocabs = [1, 2, 100, 1023, 1024, 2047, 2048, 2049, 32768, 50000, 1 << 21, 1 << 22, (1 << 22) + 1, 1 << 30, (1 << 31) - 1]
    dims = [1, 4, 5, 64, 500, 512, 513, 1024, 1025, 2048, 2049, 4096, 4100, 5000, 8192, 16384, 20001, 1 << 20]
    for v in (100, 2047, 2048, 32768):  # and every step of the chunks in one row of sizes
        for d in (512, 600, 4096):
            last = 0
            for t in range(257, 70000, 7):
                n = L.embedding_grad_workspace(t, v, d)
                assert n >= last, (t, v, d)
                last = n
    size = {(t, v, d): L.embedding_grad_workspace(t, v, d) for t in tokens for v in vocabs for d in dims}
    for (t, v, d), n in size.items():
        if t <= 256:
            assert n == 0
        else:
            assert n >= table_plan(t, v, d), (t, v, d)
    for axis in (tokens, vocabs, dims):
        for a, b in zip(axis, axis[1:]):
            for t in tokens if axis is not tokens else [None]:
                for v in vocabs if axis is not vocabs else [None]:
                    for d in dims if axis is not dims else [None]:
                        lo, hi = ((a, v, d), (b, v, d)) if t is None else ((t, a, d), (t, b, d)) if v is None else ((t, v, a), (t, v, b))
                        assert size[lo] <= size[hi], (lo, hi)
