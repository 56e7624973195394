"""More of the residual stream's operators on the GPU: calls and paths beside those of test_residual_gpu.py, whose helpers,
oracles in 64 bits and tolerances these tests use.

The depth of a column sum, which that file allows 32 + rows / 64 roundings beyond the 128 of a row's formulas, for the
split as it is: up to 256 rows a team takes one and the join of n teams adds n / 16 + 15, 31 at most.  Of more rows a team
takes two or more; n is at most rows / 2 and, for more than 1024 columns, 1280: 2 + rows / 32 + 15 roundings for up to 2560
rows are at most 25 more than the 32 + rows / 64, and fewer than those from 5000 rows on.  (Up to 1024 columns the join adds
n / 64 + 17, four teams of one wavefront having joined before it.)  A row's gradient takes about 75 of its 128: two means of
26 levels, half of that behind the square roots, and some twenty operations.
"""
import pytest

from tests.test_residual_gpu import BF, F32, PAIRS, L, backward64, gen, near, rand, sum_depth  # noqa: F401 (L is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,res", PAIRS)
@pytest.mark.parametrize("rows,dim", [(1, 1), (37, 640), (300, 1001), (5, 9000)])
def test_weight_gradient_without_a_gradient_of_the_norm(L, act, res, rows, dim):
    """No gradient reaches y: its weight's gradient is zeros, and the others are those of a call that does not ask for it."""
    import torch
    g = gen(rows + dim)
    total, h, dh = rand((rows, dim), act, g), rand((rows, dim), res, g), rand((rows, dim), res, g)
    w1, w2 = rand((dim,), act, g, 0.1, 1.0), rand((dim,), act, g, 0.1, 1.0)
    ds, dres, dw1, dw2 = torch.empty_like(total), torch.empty_like(h), torch.empty_like(w1), torch.full_like(w2, 3.0)
    L.reduce_norm_backward(h, None, dh, ds, dres, total=total, post_weight=w1, pre_weight=w2, post_weight_grad=dw1,
                           pre_weight_grad=dw2)
    assert bool((dw2 == 0).all())
    want, mag = backward64(total, None, None, dh, w1, None, None, 0, 1.0, 1e-6, 0.0, True, False)
    near(ds, want["send"], mag["send"], 256, "send")
    assert torch.equal(dres, dh)
    near(dw1, want["w1"], mag["w1"], 160, "w1")
    with pytest.raises(L.FlagcxError):  # the norm's input is needed for it
        L.reduce_norm_backward(None, None, dh, ds, dres, total=total, post_weight=w1, pre_weight=w2, pre_weight_grad=dw2)


# ------------------------------------------------- table gradient: the sorted path

def spread_tokens(rows, each, foreign, vocab, first, g):
    """ids in which `rows` rows of the table occur `each` times, shuffled, with `foreign` ids of other shards among them."""
    import torch
    named = torch.randperm(vocab, device="cuda", generator=g)[:rows] + first
    other = torch.cat([torch.randint(first - 999, first, (foreign - foreign // 2,), device="cuda", generator=g),
                       torch.randint(first + vocab, first + vocab + 999, (foreign // 2,), device="cuda", generator=g)])
    ids = torch.cat([named.repeat(each), other])
    return ids[torch.randperm(ids.numel(), device="cuda", generator=g)], named


@pytest.mark.parametrize("rows,vocab,dim,foreign", [
    (33, 1000, 70, 0), (33, 1000, 300, 57), (250, 2047, 9, 20), (250, 5 << 20, 6, 3),      # one sorting workgroup; 1, 3 passes
    (300, 700, 300, 0), (300, 5 << 20, 5, 700), (4000, 50000, 70, 1500), (4000, 50000, 520, 0),  # several; chunks of 8 to 32
    (70000, 100000, 3, 4000), (70000, 9 << 20, 4, 0)])                                     # longer than 256 tiles
def test_sorted_sums_keep_the_order_of_tokens(L, rows, vocab, dim, foreign):
    """Every row that is named holds eight tokens, spread over the batch, so each is summed whole inside one chunk of 8, 16
    or 32 sorted tokens: bit for bit the fp32 sum of its tokens from the first to the last.  Values of very different size
    tell any other order."""
    import torch
    g = gen(rows + vocab + dim)
    first = 5000
    ids, named = spread_tokens(rows, 8, foreign, vocab, first, g)
    tokens = ids.numel()
    assert tokens > 256
    grad = rand((tokens, dim), F32, g) * 2.0 ** torch.randint(-12, 13, (tokens, dim), device="cuda", generator=g)
    here = (ids >= first) & (ids < first + vocab)
    row = ids[here] - first
    order = torch.sort(row, stable=True).indices
    parts = grad[here][order].view(rows, 8, dim)
    touched = row[order].view(rows, 8)[:, 0]

    def summed(steps):
        s = parts[:, steps[0]].clone()
        for i in steps[1:]:
            s = s + parts[:, i]  # one fp32 rounding each
        return s
    want = summed(range(8))
    swapped = summed([1, 2, 0, 3, 4, 5, 6, 7])
    assert bool((swapped != want).any())  # the values do tell
    old = rand((vocab, dim), F32, g)
    for accumulate in (False, True):
        for idt in (torch.int64, torch.int32):
            table = old.clone()
            L.embedding_grad(grad, ids.to(idt), table, first=first, accumulate=accumulate)
            assert torch.equal(table[touched], want + old[touched] if accumulate else want)
            rest = torch.ones(vocab, dtype=torch.bool, device="cuda")
            rest[touched] = False
            assert torch.equal(table[rest], old[rest]) if accumulate else not bool(table[rest].any())


@pytest.mark.parametrize("tokens", [200, 700, 6000])
def test_table_of_more_than_4_gib(L, tokens):
    """Rows on both sides of 4 GiB, one of them of most tokens, written and accumulated, next to the table's clearing."""
    import torch
    if torch.cuda.get_device_properties(0).total_memory < 64 << 30:
        pytest.skip("needs memory")
    g = gen(tokens)
    vocab, dim = 70000, 32776  # row 65520 begins behind 4 GiB
    ids = torch.randint(65400, vocab + 200, (tokens,), device="cuda", generator=g)
    ids[torch.rand(tokens, device="cuda", generator=g) < 0.3] = 69999
    ids[torch.rand(tokens, device="cuda", generator=g) < 0.05] = 7
    grad = rand((tokens, dim), BF, g)
    here = ids < vocab
    named, at = torch.unique(ids[here], return_inverse=True)
    want = torch.zeros((named.numel(), dim), dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(want)
    want.index_put_((at,), grad[here].double(), accumulate=True)
    mag.index_put_((at,), grad[here].double().abs(), accumulate=True)
    rest = torch.ones(vocab, dtype=torch.bool, device="cuda")
    rest[named] = False
    table = torch.empty((vocab, dim), dtype=torch.bfloat16, device="cuda")
    for accumulate in (False, True):
        table.fill_(3.0)
        L.embedding_grad(grad, ids, table, accumulate=accumulate)
        add = 3.0 if accumulate else 0.0
        near(table[named], want + add, mag + add, sum_depth(tokens), "table")
        for part, keep in zip(table.split(10000), rest.split(10000)):
            assert bool((part[keep] == add).all())


@pytest.mark.parametrize("tokens", [0, 200, 1500, 3000])
def test_more_rows_to_clear_than_a_launch_takes(L, tokens):
    """2.3 million groups of 64 rows: clearing goes on in a second and a third launch, beside the sums of few tokens, by
    sorted keys and by flags (of which the sort's launches have cleared a million)."""
    import torch
    g = gen(tokens + 1)
    vocab = 147000011
    ids = torch.randint(-5, vocab + 5, (tokens,), device="cuda", generator=g)
    if tokens:
        ids[:4] = torch.tensor([0, vocab - 1, 64 << 20, vocab], device="cuda")
    grad = torch.ones((tokens, 1), dtype=torch.bfloat16, device="cuda")
    table = torch.full((vocab, 1), 9.0, dtype=torch.bfloat16, device="cuda")
    L.embedding_grad(grad, ids, table)
    named, count = torch.unique(ids[(ids >= 0) & (ids < vocab)], return_counts=True)
    assert torch.equal(table[named, 0].long(), count)
    assert int(torch.count_nonzero(table)) == named.numel()


def test_more_chunks_than_a_launch_takes(L):
    """134 million tokens: four million chunks and, of the short rows' joins, a second launch; whole numbers sum exactly.
    Most rows span some 40 chunks, one some 200000."""
    import torch
    if torch.cuda.get_device_properties(0).total_memory < 64 << 30:
        pytest.skip("needs memory")
    g = gen(23)
    tokens, vocab = (128 << 20) + 12345, 100003
    ids = torch.randint(0, vocab + 50, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    ids[torch.rand(tokens, device="cuda", generator=g) < 0.05] = 77
    grad = torch.randint(-8, 9, (tokens, 1), device="cuda", generator=g, dtype=torch.int8).to(torch.bfloat16)
    most = ids == 77
    want = torch.bincount(ids, weights=torch.where(most, 0.0, grad[:, 0].double()), minlength=vocab + 50)[:vocab]
    want[77] = grad[most, 0].double().sum()
    assert float(want.abs().max()) < 2 ** 23
    old = torch.arange(vocab, device="cuda", dtype=torch.float32)[:, None] % 100
    for accumulate in (False, True):
        table = old.clone()
        L.embedding_grad(grad, ids, table, accumulate=accumulate)
        assert torch.equal(table[:, 0].double(), want + (old[:, 0].double() if accumulate else 0.0))


# ------------------------------------------------------------- workspaces

def test_one_workspace_for_batches_of_many_lengths(L):
    """A workspace of the longest batch serves every shorter one, and what lies behind the size of a batch stays."""
    import torch
    g = gen(24)
    dim = 1024
    for gate_rows, longest in ((None, 300), (7, 3000), (100, 2500), (0, 700)):
        need = lambda n: L.reduce_norm_backward_workspace(n, dim, gate_rows is not None, gate_rows or 0)
        room = torch.empty(need(longest) + 256, dtype=torch.uint8, device="cuda")
        for rows in (longest, 1, 255, 256, 257, 258, 299, longest - 1):
            x, h, dy, dh = (rand((rows, dim), BF, g) for _ in range(4))
            w1, w2 = rand((dim,), BF, g, 0.1, 1.0), rand((dim,), BF, g, 0.1, 1.0)
            gate = None if gate_rows is None else rand((-(-rows // gate_rows) if gate_rows else 1, dim), BF, g)
            got = []
            for ws in (room, room[:need(rows)], None):
                room.fill_(0x5a)
                ds, dw1, dw2 = torch.empty_like(x), torch.empty_like(w1), torch.empty_like(w2)
                dg = None if gate is None else torch.empty_like(gate)
                L.reduce_norm_backward(h, dy, dh, ds, total=x, post_weight=w1, pre_weight=w2, gate=gate, gate_rows=gate_rows or 0,
                                       post_weight_grad=dw1, pre_weight_grad=dw2, gate_grad=dg, workspace=ws)
                assert bool((room[need(rows):] == 0x5a).all())
                got.append([ds, dw1, dw2] + ([] if dg is None else [dg]))
            assert all(torch.equal(a, b) for other in got[1:] for a, b in zip(got[0], other)), (rows, gate_rows)


def test_one_workspace_for_table_gradients_of_many_sizes(L):
    import torch
    g = gen(25)
    need = L.embedding_grad_workspace
    room = torch.empty(need(33000, 2100, 520) + 256, dtype=torch.uint8, device="cuda")
    for tokens, vocab, dim in ((33000, 2100, 520), (32769, 2048, 512), (32777, 2047, 512), (2049, 2047, 64), (2048, 100, 513),
                               (8193, 2048, 520), (257, 2100, 520), (256, 2100, 520), (30, 5, 7)):
        ids = torch.randint(0, vocab, (tokens,), device="cuda", generator=g)
        grad = rand((tokens, dim), BF, g)
        tables = []
        for ws in (room, room[:need(tokens, vocab, dim)], None):
            room.fill_(0x5a)
            tables.append(L.embedding_grad(grad, ids, torch.full((vocab, dim), 4.0, device="cuda"), workspace=ws))
            assert bool((room[need(tokens, vocab, dim):] == 0x5a).all())
        assert torch.equal(tables[0], tables[1]) and torch.equal(tables[0], tables[2]), (tokens, vocab, dim)
