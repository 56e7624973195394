"""CPU checks of the residual stream's entry points: what they refuse before they touch a device, what they accept
without work, and their workspace sizes."""
import ctypes as C

import pytest

from flagcx_amd import local as L

INV = int(L.Result.InvalidArgument)
BF, F16, F32 = 9, 6, 7
P = 1 << 20  # made-up device addresses, far apart; nothing here reaches a launch


def at(n):
    return P + (n << 32)


def end(rows=4, dim=64, norms=3, act=BF, res=BF, weight=BF, scale=1.0, eps=1e-6, offset=0.0, w1=at(20), w2=at(21), gate=None,
        gatestride=0, gaterows=0):
    return L.BlockEnd(rows, dim, norms, act, res, weight, scale, eps, offset, w1, w2, gate, gatestride, gaterows)


def forward(e, srcs=(at(1), at(2)), n=None, sstride=0, res=at(3), rstride=0, out=at(4), ostride=0, norm=at(5), nstride=0,
            total=at(6), tstride=0):
    arr = (C.c_void_p * max(len(srcs), 1))(*srcs)
    st = L.Stream(None)
    return L.lib().flagcxLocalReduceNorm(e, arr, len(srcs) if n is None else n, sstride, res, rstride, out, ostride, norm,
                                         nstride, total, tstride, C.byref(st))


def backward(e, total=at(1), h=at(2), dy=at(3), dh=at(4), ds=at(5), dres=at(6), dw1=at(7), dw2=at(8), dg=None, ws=at(9),
             wbytes=1 << 31, strides=(0, 0, 0, 0, 0, 0, 0)):
    st = L.Stream(None)
    return L.lib().flagcxLocalReduceNormBackward(e, total, strides[0], h, strides[1], dy, strides[2], dh, strides[3], ds,
                                                 strides[4], dres, strides[5], dw1, dw2, dg, strides[6], ws, wbytes, C.byref(st))


def text():
    return L.lib().flagcxLocalGetLastError().decode()


@pytest.mark.parametrize("bad,word", [
    (dict(act=2), "data type"), (dict(act=10), "data type"), (dict(act=F16, res=BF), "residualtype"),
    (dict(act=F32, res=BF), "residualtype"), (dict(weight=F16), "weighttype"), (dict(norms=4), "norms"),
    (dict(norms=-1), "norms"), (dict(dim=0), "dim"), (dict(dim=16385), "dim"), (dict(eps=0.0), "eps"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(rows=1 << 41), "rows"),
])
def test_block_end_is_checked_in_both_directions(bad, word):
    assert forward(end(**bad)) == INV and word in text()
    assert backward(end(**bad)) == INV and word in text()
    n = C.c_size_t()
    assert L.lib().flagcxLocalReduceNormBackwardWorkspace(end(**bad), C.byref(n)) == INV and word in text()


def test_forward_refusals():
    assert forward(None) == INV
    assert forward(end(), n=0) == INV and "nranks" in text()
    assert forward(end(), srcs=[at(1)] * 65) == INV and "nranks" in text()
    assert forward(end(), srcs=(at(1), None)) == INV and "sendbuffs[1]" in text()
    assert forward(end(), out=None) == INV and "residualout" in text()
    assert forward(end(), norm=None) == INV and "normout" in text()
    assert forward(end(norms=1)) == INV and "normout" in text()             # normout without the norm
    assert forward(end(), srcs=(at(1), at(2) + 1)) == INV and "aligned" in text()
    assert forward(end(res=F32), out=at(4) + 2) == INV and "aligned" in text()
    assert forward(end(), sstride=63) == INV and "stride" in text()
    assert forward(end(), ostride=63) == INV and "stride" in text()
    assert forward(end(gate=at(7), gaterows=2, gatestride=5)) == INV and "stride" in text()
    assert forward(end(rows=1 << 39), ostride=1 << 40) == INV and "overflows" in text()
    st = C.byref(L.Stream(None))
    assert L.lib().flagcxLocalReduceNorm(end(), None, 2, 0, None, 0, at(4), 0, at(5), 0, None, 0, st) == INV


def test_forward_overlaps():
    row = 64 * 2
    assert forward(end(), out=at(1) + row) == INV and "overlaps" in text()  # shifted by a row
    assert forward(end(), out=at(1), ostride=72) == INV and "overlaps" in text()  # same address, other stride
    assert forward(end(res=F32), out=at(1)) == INV and "overlaps" in text()  # same address, other type
    assert forward(end(), norm=at(4)) == INV and "overlaps" in text()       # two outputs
    assert forward(end(), total=at(4) + 3 * row) == INV and "overlaps" in text()
    assert forward(end(), out=at(20) - row) == INV and "overlaps" in text()  # a weight in the output's last rows
    assert forward(end(gate=at(4), gaterows=1)) == INV and "overlaps" in text()  # gates are never written over
    # the last source alone is in the way
    assert forward(end(), srcs=[at(1)] * 63 + [at(4) + row]) == INV and "overlaps" in text()


def test_forward_side_by_side_in_one_stride_is_no_overlap():
    # residualout and normout interleaved in rows of 128 elements pass; one element closer they do not
    bad = end(rows=4, dim=64, eps=0.0)
    assert forward(bad) == INV and "eps" in text()
    e = end(rows=4, dim=64)
    assert forward(e, out=at(4), ostride=128, norm=at(4) + 63 * 2, nstride=128) == INV and "overlaps" in text()
    assert forward(e, out=at(4), ostride=128, norm=at(4) + 64 * 2, nstride=128, total=at(4) + 100 * 2, tstride=128) == INV
    assert "sumout overlaps" in text() or "overlaps sumout" in text()       # and not the pair before it


def test_backward_refusals():
    assert backward(None) == INV
    assert backward(end(), dy=None, dh=None) == INV and "NULL" in text()
    assert backward(end(), h=None) == INV and "residualout" in text()
    assert backward(end(), total=None) == INV and "sum" in text()
    assert backward(end(norms=2, gate=at(10)), dw1=None, total=None, dg=at(11)) == INV and "sum" in text()
    assert backward(end(norms=1), dy=at(3)) == INV and ("preweightgrad" in text() or "normgrad" in text())
    assert backward(end(norms=2), dw1=at(7)) == INV and "postweightgrad" in text()
    assert backward(end(w2=None)) == INV and "preweightgrad" in text()
    assert backward(end(), dg=at(11)) == INV and "gategrad" in text()
    assert backward(end(), ws=None) == INV and "workspace" in text()
    assert backward(end(), ws=at(9) + 8) == INV and "aligned" in text()
    n = C.c_size_t()
    assert L.lib().flagcxLocalReduceNormBackwardWorkspace(end(), C.byref(n)) == 0 and n.value > 0
    assert backward(end(), wbytes=n.value - 1) == INV and "needed" in text()
    assert backward(end(), ws=at(4), wbytes=n.value) == INV and "overlaps" in text()
    assert backward(end(), ds=at(4) + 128) == INV and "overlaps" in text()
    assert backward(end(), dw1=at(8)) == INV and "overlaps" in text()
    assert backward(end(), dw2=at(21)) == INV and "overlaps" in text()      # over the weight itself
    assert backward(end(gate=at(10), gaterows=1), dg=at(10)) == INV and "overlaps" in text()
    assert backward(end(), strides=(0, 63, 0, 0, 0, 0, 0)) == INV and "stride" in text()


def test_groups_of_more_rows_than_any_matrix_are_checked_like_others():
    for n in (5, 1 << 40, (1 << 64) - 1):
        assert forward(end(gate=at(7) + 1, gaterows=n)) == INV and "gate not aligned" in text()
        assert backward(end(gate=at(7) + 1, gaterows=n)) == INV and "gate not aligned" in text()
        assert forward(end(gate=at(4), gaterows=n)) == INV and "overlaps gate" in text()


def test_nothing_to_do():
    assert forward(end(rows=0)) == 0
    lib, st = L.lib(), C.byref(L.Stream(None))
    assert lib.flagcxLocalEmbedding(None, BF, 0, 64, 0, None, 4, 0, 0, 1.0, None, BF, 0, st) == 0
    assert lib.flagcxLocalEmbeddingGrad(None, BF, 0, None, 4, 0, 0, 1.0, None, BF, 10, 64, 0, 1, None, 0, st) == 0
    assert lib.flagcxLocalEmbeddingGrad(None, BF, 0, None, 4, 5, 0, 1.0, None, BF, 0, 64, 0, 0, None, 0, st) == 0


def lookup(table=at(1), tt=BF, vocab=10, dim=64, tstride=0, ids=at(2), it=4, tokens=5, out=at(3), ot=BF, ostride=0):
    return L.lib().flagcxLocalEmbedding(table, tt, vocab, dim, tstride, ids, it, tokens, 0, 1.0, out, ot, ostride,
                                        C.byref(L.Stream(None)))


def gradient(grad=at(1), ot=BF, gstride=0, ids=at(2), it=4, tokens=600, table=at(3), tt=BF, vocab=10, dim=64, tstride=0, acc=0,
             ws=at(4), wbytes=1 << 30):
    return L.lib().flagcxLocalEmbeddingGrad(grad, ot, gstride, ids, it, tokens, 0, 1.0, table, tt, vocab, dim, tstride, acc,
                                            ws, wbytes, C.byref(L.Stream(None)))


def test_embedding_refusals():
    for kw, word in [(dict(tt=2), "tabletype"), (dict(ot=0), "outtype"), (dict(tt=F16, ot=BF), "outtype"),
                     (dict(it=1), "idtype"), (dict(it=7), "idtype"), (dict(table=None), "NULL"), (dict(ids=None), "NULL"),
                     (dict(out=None), "NULL"), (dict(out=at(3) + 1), "aligned"), (dict(ids=at(2) + 4), "aligned"),
                     (dict(tstride=63), "stride"), (dict(ostride=63), "stride"), (dict(dim=1 << 31), "too large"),
                     (dict(out=at(1) + 128), "overlaps"), (dict(out=at(2)), "overlaps"), (dict(out=at(1)), "overlaps")]:
        assert lookup(**kw) == INV and word in text(), kw


def test_embedding_grad_refusals():
    n = L.embedding_grad_workspace(600, 10, 64)
    assert n > 0
    for kw, word in [(dict(tt=4), "tabletype"), (dict(ot=0), "outtype"), (dict(tt=F16, ot=BF), "outtype"),
                     (dict(it=5), "idtype"), (dict(table=None), "NULL"), (dict(ids=None), "NULL"), (dict(grad=None), "NULL"),
                     (dict(ws=None), "workspace"), (dict(ws=at(4) + 4), "aligned"), (dict(wbytes=n - 1), "needed"),
                     (dict(tokens=1 << 31), "too large"), (dict(vocab=1 << 31), "too large"), (dict(tstride=63), "stride"),
                     (dict(table=at(1)), "overlaps"), (dict(ws=at(3), wbytes=n), "overlaps"),
                     (dict(ws=at(1), wbytes=n), "overlaps")]:
        assert gradient(**kw) == INV and word in text(), kw


def test_workspace_sizes():
    n = C.c_size_t()
    lib = L.lib()
    assert lib.flagcxLocalEmbeddingGradWorkspace(5, 10, 64, None) == INV
    assert lib.flagcxLocalReduceNormBackwardWorkspace(end(), None) == INV
    assert lib.flagcxLocalReduceNormBackwardWorkspace(None, C.byref(n)) == INV
    assert L.embedding_grad_workspace(0, 10, 64) == 0 and L.embedding_grad_workspace(900, 0, 64) == 0
    assert L.embedding_grad_workspace(256, 10, 64) == 0 < L.embedding_grad_workspace(257, 10, 64)
    assert gradient(tokens=256, ws=None, wbytes=0, acc=1, table=at(1)) == INV and "overlaps" in text()  # and not a workspace
    # the sums' partial rows stay below the rows that they stand for, however many there are
    for rows in (1, 7, 64, 1000, 16384, 1 << 20):
        for dim in (1, 64, 1000, 8192, 16384):
            for gate_rows in (0, 1, 2, 5, 100, 4096, 1 << 22):
                b = L.reduce_norm_backward_workspace(rows, dim, True, gate_rows)
                assert b <= 3 * 4 * dim * (rows // 2 + 16385) and b % (12 * dim) == 0, (rows, dim, gate_rows)
                assert b // (12 * dim) <= max(1, rows), (rows, dim, gate_rows)
    assert L.reduce_norm_backward_workspace(0, 64) == 0


def test_python_binding_refuses_host_tensors():
    import torch
    x = torch.zeros(4, 8)
    for call in (lambda: L.reduce_norm([x], x, x, x), lambda: L.reduce_norm([], x, x, x),
                 lambda: L.reduce_norm_backward(x, x, x, x, x, total=x),
                 lambda: L.reduce_norm_backward(None, None, None),
                 lambda: L.embedding(x, torch.zeros(3, dtype=torch.int64), x), lambda: L.embedding_grad(x, x, x)):
        with pytest.raises(L.FlagcxError) as e:
            call()
        assert e.value.code == INV
