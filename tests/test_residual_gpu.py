"""The residual stream's operators on the GPU against their definitions in 64 bits.

Tolerances, element by element.  A result that is rounded once is off by half a step, eps/2 of its type relative to the
value (and by half the smallest subnormal of fp16 near zero).  Before it the arithmetic is fp32: a value formed of terms
t_1 .. t_n by D roundings is off by at most D * 2^-24 * sum |t_i|, and the terms' absolute values are carried through the
same formula as the values themselves (`mag`).  D for the rows' formulas: a fold of up to 64 inputs (64), a mean over a
row (up to 16 products in a lane, 10 levels over lanes and wavefronts; half of that after the square root) and about ten
operations an element: 128 covers them.  Column sums add the rows that one team takes and the join of the teams: a team
takes at most max(4, rows / 256) rows here, the join teams / 16 + 16: with rows / 4 teams, rows / 64 + 32 more.  (Where the
join takes sixteen columns to a wavefront it is teams / 64 + 18 and, before it, 4 for teams that share a workgroup.)
"""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, F16, F32 = "bfloat16", "float16", "float32"
PAIRS = [(BF, BF), (BF, F32), (F16, F16), (F16, F32), (F32, F32)]


@pytest.fixture(scope="module")
def L():
    import torch
    assert torch.cuda.is_available()
    from flagcx_amd import local
    assert local.lib().flagcxLocalInit() == 0
    return local


def dt(name):
    import torch
    return getattr(torch, name)


def gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(shape, dtype, g, mul=1.0, add=0.0):
    import torch
    return (torch.randn(shape, device="cuda", generator=g, dtype=torch.float32) * mul + add).to(dt(dtype))


def wide(rows, dim, pad, dtype, g, mul=1.0, fill=None, shift=0):
    """A rows x dim view of rows that are `pad` elements longer, `shift` elements into its allocation; with the allocation."""
    import torch
    full = torch.empty(rows * (dim + pad) + shift + 8, dtype=dt(dtype), device="cuda")
    if fill is not None:
        full.fill_(fill)
    view = full[shift:shift + rows * (dim + pad)].view(rows, dim + pad)[:, :dim]
    if fill is None:
        full.fill_(7.0)
        view.copy_(rand((rows, dim), dtype, g, mul))
    return view, full


def near(got, want, mag, depth, what):
    import torch
    want = want.to(torch.float64)
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + depth * U * mag * 1.01 + tiny
    off = (got.to(torch.float64) - want).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((off / tol.clamp_min(1e-300)).max()), got.shape)


def gates_of_rows(gate, gate_rows, rows):
    if gate is None:
        return None
    g = gate.double()
    if gate_rows == 0:
        return g.reshape(1, -1).expand(rows, -1)
    return g.repeat_interleave(gate_rows, 0)[:rows]


def forward64(srcs, residual, w1, w2, gate, gate_rows, scale, eps, offset, post):
    """(s, h, y) and their magnitudes."""
    import torch
    rows, dim = srcs[0].shape
    s = sum(x.double() for x in srcs)
    ms = sum(x.double().abs() for x in srcs)
    u, mu = s, ms
    if post:
        r1 = (s.square().mean(1, keepdim=True) + eps) ** -0.5
        f1 = r1 if w1 is None else r1 * (w1.double() + offset)
        m1 = r1 if w1 is None else r1 * (w1.double().abs() + abs(offset))
        u, mu = s * f1, ms * m1
    g = gates_of_rows(gate, gate_rows, rows)
    if g is not None:
        u, mu = u * g, mu * g.abs()
    h = scale * u
    mh = abs(scale) * mu
    if residual is not None:
        h, mh = h + residual.double(), mh + residual.double().abs()
    r2 = (h.square().mean(1, keepdim=True) + eps) ** -0.5
    f2 = r2 if w2 is None else r2 * (w2.double() + offset)
    m2 = r2 if w2 is None else r2 * (w2.double().abs() + abs(offset))
    # an error of h also moves r2, by at most the row's relative error
    rel = (mh * h.abs()).mean(1, keepdim=True) / (h.square().mean(1, keepdim=True) + eps)
    return (s, h, h * f2), (ms, mh, mh * m2 + (h * m2).abs() * rel)


def backward64(total, h, dy, dh, w1, w2, gate, gate_rows, scale, eps, offset, post, pre):
    import torch
    ref = total if total is not None else h if h is not None else dh
    rows, dim = ref.shape
    zero = torch.zeros((rows, dim), dtype=torch.float64, device="cuda")
    d = dh.double() if dh is not None else zero
    md = d.abs()
    out, mag = {}, {}
    if pre:
        y = dy.double() if dy is not None else zero
        q = (h.double().square().mean(1, keepdim=True) + eps) ** -0.5
        n2 = h.double() * q
        wy = y if w2 is None else y * (w2.double() + offset)
        my = y.abs() if w2 is None else y.abs() * (w2.double().abs() + abs(offset))
        d = d + q * (wy - n2 * (wy * n2).mean(1, keepdim=True))
        md = md + q * (my + n2.abs() * (my * n2.abs()).mean(1, keepdim=True))
        out["w2"], mag["w2"] = (y * n2).sum(0), (y * n2).abs().sum(0)
    out["res"], mag["res"] = d, md
    u = mu = None
    if total is not None:
        s = total.double()
        u, mu = s, s.abs()
        if post:
            r = (s.square().mean(1, keepdim=True) + eps) ** -0.5
            n1 = s * r
            f1 = 1.0 if w1 is None else w1.double() + offset
            m1 = 1.0 if w1 is None else w1.double().abs() + abs(offset)
            u, mu = n1 * f1, n1.abs() * m1
    g = gates_of_rows(gate, gate_rows, rows)
    c, mc = scale * d, abs(scale) * md
    if g is not None and u is not None:
        def joined(x):
            if gate_rows == 0:
                return x.sum(0)
            return torch.stack([p.sum(0) for p in x.split(gate_rows)])
        out["gate"], mag["gate"] = joined(c * u), joined(mc * mu)
    if g is not None:
        c, mc = c * g, mc * g.abs()
    if post:
        out["w1"], mag["w1"] = (c * n1).sum(0), (mc * n1.abs()).sum(0)
        c, mc = c * f1, mc * m1
        c = r * (c - n1 * (c * n1).mean(1, keepdim=True))
        mc = r * (mc + n1.abs() * (mc * n1.abs()).mean(1, keepdim=True))
    out["send"], mag["send"] = c, mc
    return out, mag


# ------------------------------------------------------------------ forward

FWD = [  # ranks, rows, dim, pad, shift, post, gate_rows (None: no gate), weight fp32, offset, sum
    (1, 1, 1, 0, 0, True, 0, False, 0.0, True),
    (2, 3, 5, 0, 0, True, None, True, 1.0, True),
    (3, 70, 64, 0, 0, False, 1, False, 0.0, False),
    (8, 9, 512, 0, 0, True, 4, True, 0.0, True),
    (9, 7, 520, 8, 0, True, 0, False, 1.0, True),
    (64, 2, 129, 3, 1, True, 3, False, 0.0, True),
    (5, 13, 1024, 64, 0, False, None, False, 0.0, False),
    (4, 6, 2047, 0, 0, True, 2, True, 0.5, True),
    (7, 5, 4096, 0, 1, True, 0, False, 0.0, True),
    (3, 4, 8192, 0, 0, True, 3, False, 0.0, True),
    (6, 3, 8193, 1, 0, True, 1, True, 1.0, True),
    (3, 2, 16384, 0, 0, True, 0, False, 0.0, True),
    (2, 2, 16383, 0, 3, False, None, True, 0.0, False),
    (3, 19, 8, 1, 5, True, 2, False, 0.0, True),     # rows that start anywhere inside vectors, but all alike
    (2, 21, 9, 0, 0, True, 1, True, 1.0, True),
    (5, 17, 1003, 2, 0, True, 4, False, 0.0, True),
    (2, 9, 8189, 0, 3, True, 0, True, 0.0, True),
    (2, 1031, 5001, 0, 1, True, None, False, 0.5, True),
    (1, 5, 16377, 0, 0, True, 0, False, 0.0, False),
    (15, 6, 128, 0, 0, True, 2, False, 0.0, True),   # every remainder of inputs, at every length of a lane's share
    (31, 3, 256, 0, 0, True, None, True, 0.0, True),
    (14, 4, 99, 0, 0, False, 0, False, 0.0, True),
    (15, 3, 264, 0, 0, True, None, False, 0.0, True),
    (15, 600, 4200, 0, 0, False, None, False, 0.0, True),
    (7, 600, 4201, 0, 0, False, None, False, 0.0, True),
]


@pytest.mark.parametrize("act,res", PAIRS)
@pytest.mark.parametrize("case", FWD, ids=lambda c: "k%d_%dx%d" % c[:3])
def test_forward(L, act, res, case):
    import torch
    ranks, rows, dim, pad, shift, post, gate_rows, f32w, offset, keep = case
    g = gen(ranks * 1000 + dim)
    scale, eps = 0.75, 1e-5
    srcs = [wide(rows, dim, pad, act, g, 1.0, shift=shift)[0] for _ in range(ranks)]
    residual = wide(rows, dim, pad, res, g, 2.0, shift=shift)[0]
    wt = F32 if f32w else act
    w1, w2 = rand((dim,), wt, g, 0.2, 1 - offset), rand((dim,), wt, g, 0.2, 1 - offset)
    if not post:
        w1 = None
    gate = None if gate_rows is None else \
        rand((dim,) if gate_rows == 0 else (-(-rows // gate_rows), dim), act, g, 0.5, 0.5)
    out, out_full = wide(rows, dim, pad, res, g, fill=5.0, shift=shift)
    y, y_full = wide(rows, dim, pad, act, g, fill=5.0, shift=shift)
    s, s_full = wide(rows, dim, pad, act, g, fill=5.0, shift=shift) if keep else (None, None)
    L.reduce_norm(srcs, residual, out, y, sum_out=s, post_weight=w1, pre_weight=w2, gate=gate, gate_rows=gate_rows or 0,
                  scale=scale, eps=eps, weight_offset=offset)
    (ws, wh, wy), (ms, mh, my) = forward64(srcs, residual, w1, w2, gate, gate_rows or 0, scale, eps, offset, post)
    near(out, wh, mh, 128, "stream")
    near(y, wy, my, 128, "norm")
    if keep:
        near(s, ws, ms, 64, "sum")
    for view, full in ((out, out_full), (y, y_full), (s, s_full)):  # nothing between and around the rows
        if full is not None:
            view.fill_(5.0)
            assert bool((full == 5.0).all())


@pytest.mark.parametrize("act,res", PAIRS)
def test_forward_without_the_optional_parts(L, act, res):
    """No residual, no weights, a norm on one side, the other or none; the sum equals the plain fold bit for bit."""
    import torch
    g = gen(5)
    rows, dim, ranks = 11, 768, 4
    srcs = [rand((rows, dim), act, g) for _ in range(ranks)]
    plain = torch.empty((rows, dim), dtype=dt(act), device="cuda")
    L.reduce(srcs, plain, L.RedOp.Sum)
    for post in (False, True):
        for pre in (False, True):
            out = torch.empty((rows, dim), dtype=dt(res), device="cuda")
            y = torch.empty((rows, dim), dtype=dt(act), device="cuda") if pre else None
            s = torch.empty((rows, dim), dtype=dt(act), device="cuda")
            L.reduce_norm(srcs, None, out, y, sum_out=s, post_norm=post, eps=1e-6)
            (_, wh, wy), (_, mh, my) = forward64(srcs, None, None, None, None, 0, 1.0, 1e-6, 0.0, post)
            near(out, wh, mh, 128, "stream")
            if pre:
                near(y, wy, my, 128, "norm")
            assert torch.equal(s, plain)
            if not post and act == res:
                assert torch.equal(out, plain)


def test_forward_in_place(L):
    """The stream over itself, the norm over a source, the sum over another."""
    import torch
    g = gen(6)
    for rows, dim in ((5, 512), (3, 1537), (2, 10000)):
        srcs = [rand((rows, dim), BF, g) for _ in range(3)]
        residual, w1, w2 = rand((rows, dim), F32, g), rand((dim,), BF, g, 0.1, 1.0), rand((dim,), BF, g, 0.1, 1.0)
        out, y, s = (torch.empty((rows, dim), dtype=dt(d), device="cuda") for d in (F32, BF, BF))
        L.reduce_norm(srcs, residual, out, y, sum_out=s, post_weight=w1, pre_weight=w2)
        a = [x.clone() for x in srcs]
        r = residual.clone()
        L.reduce_norm(a, r, r, a[0], sum_out=a[2], post_weight=w1, pre_weight=w2)
        assert torch.equal(r, out) and torch.equal(a[0], y) and torch.equal(a[2], s) and torch.equal(a[1], srcs[1])


def test_forward_rows_keep_to_themselves(L):
    """NaN, infinities and zeros in one row leave the others bit for bit alone; a row of zeros gives zeros."""
    import torch
    g = gen(7)
    for dim in (33, 512, 1024, 8193):
        rows = 9
        srcs = [rand((rows, dim), F16, g) for _ in range(2)]
        residual, w = rand((rows, dim), F16, g), rand((dim,), F16, g, 0.1, 1.0)
        out, y, out2, y2 = (torch.empty((rows, dim), dtype=dt(F16), device="cuda") for _ in range(4))
        L.reduce_norm(srcs, residual, out, y, post_weight=w, pre_weight=w)
        srcs[0][1, 0] = float("nan")
        srcs[0][3, dim - 1] = float("inf")
        srcs[0][5], srcs[1][5], residual[5] = 0.0, 0.0, 0.0
        L.reduce_norm(srcs, residual, out2, y2, post_weight=w, pre_weight=w)
        for r in range(rows):
            if r == 1:
                assert bool(out2[r].isnan().all()) and bool(y2[r].isnan().all())
            elif r == 3:  # inf / inf where the infinity stands, the rest of the block's result is zero
                assert bool(out2[r, dim - 1].isnan()) and bool(y2[r].isnan().all())
            elif r == 5:
                assert bool((out2[r] == 0).all()) and bool((y2[r] == 0).all())
            else:
                assert torch.equal(out[r], out2[r]) and torch.equal(y[r], y2[r])


# ----------------------------------------------------------------- backward

BWD = [  # rows, dim, pad, shift, post, pre, gate_rows, weight fp32, offset
    (1, 1, 0, 0, True, True, 0, False, 0.0),
    (3, 7, 0, 0, True, True, None, True, 1.0),
    (70, 64, 0, 0, False, True, 1, False, 0.0),
    (513, 96, 0, 0, True, True, 7, True, 0.0),
    (300, 512, 8, 0, True, True, 100, False, 1.0),
    (41, 520, 0, 0, True, False, 0, False, 0.0),
    (517, 1535, 0, 0, True, True, 1, True, 0.0),
    (33, 2048, 0, 0, True, True, 2, False, 0.0),
    (5, 4096, 0, 1, True, True, 3, False, 0.0),
    (19, 8192, 0, 0, True, True, 0, True, 0.5),
    (11, 8195, 5, 0, True, True, 4, False, 0.0),
    (9, 16384, 0, 0, True, True, 0, False, 0.0),
    (6, 16381, 0, 0, True, True, 1, True, 1.0),
    (10, 16384, 0, 0, True, True, 9, False, 0.0),
    (1030, 640, 0, 0, False, False, 5, False, 0.0),
    (9000, 48, 0, 0, True, True, 2, True, 0.0),
    (9001, 512, 0, 0, True, True, 1, False, 0.0),  # four teams of one wavefront to a workgroup, the last not full
    (8195, 264, 8, 0, True, True, None, True, 1.0),
    (9003, 96, 0, 0, True, True, 4001, False, 0.0),
    (9002, 131, 0, 1, True, True, 0, True, 0.0),
    (2100, 1000, 0, 0, True, True, 700, False, 0.0),
    (9, 8, 1, 5, True, True, 2, False, 0.0),  # rows that start anywhere inside vectors, but all alike
    (300, 9, 0, 0, True, True, 1, True, 1.0),
    (1029, 1003, 2, 0, True, True, 500, False, 0.0),
    (270, 5001, 0, 3, True, True, 0, True, 0.0),
    (23, 8187, 0, 0, True, True, None, False, 0.5),
    (261, 9001, 0, 0, True, True, 1, False, 0.0),
    (265, 16377, 4, 1, True, True, 130, False, 0.0),
    (5000, 77, 0, 0, True, True, 0, False, 0.0),
    (60, 333, 0, 0, True, True, 3, False, 0.0),
    (900, 6144, 0, 0, True, True, 100, True, 0.0),  # groups in turns, of several teams or of one, the last one shorter
    (1300, 4104, 0, 0, True, True, 7, False, 0.0),
    (777, 9000, 0, 0, True, True, 260, False, 0.0),
    (1111, 5001, 0, 3, False, True, 301, False, 0.0),
    (6000, 513, 0, 0, True, True, 11, False, 1.0),
    (8300, 64, 0, 0, True, False, 4099, True, 0.0),
]


@pytest.mark.parametrize("act,res", PAIRS)
@pytest.mark.parametrize("case", BWD, ids=lambda c: "%dx%d_g%s" % (c[0], c[1], c[6]))
def test_backward(L, act, res, case):
    import torch
    rows, dim, pad, shift, post, pre, gate_rows, f32w, offset = case
    g = gen(rows * 31 + dim)
    scale, eps = 0.75, 1e-5
    total, h = wide(rows, dim, pad, act, g, shift=shift)[0], wide(rows, dim, pad, res, g, 2.0, shift=shift)[0]
    dy = wide(rows, dim, pad, act, g, 0.1, shift=shift)[0] if pre else None
    dh = wide(rows, dim, pad, res, g, 0.1, shift=shift)[0]
    wt = F32 if f32w else act
    w1 = rand((dim,), wt, g, 0.2, 1 - offset) if post else None
    w2 = rand((dim,), wt, g, 0.2, 1 - offset) if pre else None
    gate = None if gate_rows is None else \
        rand((dim,) if gate_rows == 0 else (-(-rows // gate_rows), dim), act, g, 0.5, 0.5)
    ds, ds_full = wide(rows, dim, pad, act, g, fill=5.0, shift=shift)
    dres, dres_full = wide(rows, dim, pad, res, g, fill=5.0, shift=shift)
    dw1 = torch.full((dim,), 5.0, dtype=dt(wt), device="cuda") if post else None
    dw2 = torch.full((dim,), 5.0, dtype=dt(wt), device="cuda") if pre else None
    dg = None if gate is None else torch.full_like(gate, 5.0)
    args = dict(total=total, post_weight=w1, pre_weight=w2, gate=gate, gate_rows=gate_rows or 0, scale=scale, eps=eps,
                weight_offset=offset)
    L.reduce_norm_backward(h, dy, dh, ds, dres, post_weight_grad=dw1, pre_weight_grad=dw2, gate_grad=dg, **args)
    want, mag = backward64(total, h, dy, dh, w1, w2, gate, gate_rows or 0, scale, eps, offset, post, pre)
    deep = 128 + rows // 64 + 32
    near(ds, want["send"], mag["send"], 256, "send")      # two formulas in a row
    near(dres, want["res"], mag["res"], 128, "res")
    if post:
        near(dw1, want["w1"], mag["w1"], deep, "w1")
    if pre:
        near(dw2, want["w2"], mag["w2"], deep, "w2")
    if gate is not None:
        near(dg, want["gate"].reshape(dg.shape), mag["gate"].reshape(dg.shape), deep, "gate")
    # the same call again gives the same bits, and each gradient alone is the one of all together
    again = [None if t is None else torch.full_like(t, 3.0) for t in (ds, dres, dw1, dw2, dg)]
    L.reduce_norm_backward(h, dy, dh, again[0], again[1], post_weight_grad=again[2], pre_weight_grad=again[3],
                           gate_grad=again[4], **args)
    names = ("send_grad", "residual_grad", "post_weight_grad", "pre_weight_grad", "gate_grad")
    for i, (a, b) in enumerate(zip((ds, dres, dw1, dw2, dg), again)):
        if a is not None:
            assert torch.equal(a, b), names[i]
            alone = torch.full_like(a, 3.0)
            L.reduce_norm_backward(h, dy, dh, **{names[i]: alone}, **args)
            assert torch.equal(a, alone), names[i] + " alone"
    for view, full in ((ds, ds_full), (dres, dres_full)):
        view.fill_(5.0)
        assert bool((full == 5.0).all())


def test_backward_with_one_gradient_missing_and_in_place(L):
    import torch
    g = gen(8)
    for rows, dim in ((37, 640), (4, 9000)):
        total, h, dy, dh = (rand((rows, dim), BF, g) for _ in range(4))
        w1, w2 = rand((dim,), BF, g, 0.1, 1.0), rand((dim,), BF, g, 0.1, 1.0)
        ds, dres, dw2 = torch.empty_like(dh), torch.empty_like(dh), torch.empty_like(w2)
        L.reduce_norm_backward(h, dy, None, ds, dres, total=total, post_weight=w1, pre_weight=w2, pre_weight_grad=dw2)
        want, mag = backward64(total, h, dy, None, w1, w2, None, 0, 1.0, 1e-6, 0.0, True, True)
        near(ds, want["send"], mag["send"], 256, "send")
        near(dres, want["res"], mag["res"], 128, "res")
        near(dw2, want["w2"], mag["w2"], 192, "w2")
        L.reduce_norm_backward(None, None, dh, ds, dres, total=total, post_weight=w1)
        want, mag = backward64(total, None, None, dh, w1, None, None, 0, 1.0, 1e-6, 0.0, True, False)
        near(ds, want["send"], mag["send"], 256, "send")
        assert torch.equal(dres, dh)
        L.reduce_norm_backward(h, dy, dh, ds, dres, total=total, post_weight=w1, pre_weight=w2)
        a, b = dy.clone(), dh.clone()
        L.reduce_norm_backward(h, a, b, a, b, total=total, post_weight=w1, pre_weight=w2)
        assert torch.equal(a, ds) and torch.equal(b, dres)
        a, b = total.clone(), h.clone()
        L.reduce_norm_backward(b, dy, dh, a, b, total=a, post_weight=w1, pre_weight=w2)
        assert torch.equal(a, ds) and torch.equal(b, dres)


@pytest.mark.parametrize("rows,dim", [(37, 640), (9, 1001), (4, 9000), (3, 8201)])
def test_every_output_over_every_input(L, rows, dim):
    """Each output in the place of each input that it may replace gives the bits of separate buffers."""
    import torch
    g = gen(rows + dim)
    w, gate = rand((dim,), BF, g, 0.1, 1.0), rand((rows, dim), BF, g, 0.3, 0.5)
    ins = {k: rand((rows, dim), BF, g) for k in ("total", "h", "dy", "dh")}

    def backward(b):
        L.reduce_norm_backward(b["h"], b["dy"], b["dh"], b["ds"], b["dres"], total=b["total"], post_weight=w, pre_weight=w,
                               gate=gate, gate_rows=1)
        return b["ds"].clone(), b["dres"].clone()

    want = backward({**ins, "ds": torch.empty_like(gate), "dres": torch.empty_like(gate)})
    for over in ins:
        for out in ("ds", "dres"):
            b = {k: v.clone() for k, v in ins.items()}
            b.update(ds=torch.empty_like(gate), dres=torch.empty_like(gate))
            b[out] = b[over]
            got = backward(b)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (out, over)

    ins = {k: rand((rows, dim), BF, g) for k in ("a", "b", "residual")}

    def forward(b):
        L.reduce_norm([b["a"], b["b"]], b["residual"], b["out"], b["y"], sum_out=b["s"], post_weight=w, pre_weight=w,
                      gate=gate, gate_rows=1)
        return [b[k].clone() for k in ("out", "y", "s")]

    want = forward({**ins, **{k: torch.empty_like(gate) for k in ("out", "y", "s")}})
    for over in ins:
        for out in ("out", "y", "s"):
            b = {k: v.clone() for k, v in ins.items()}
            b.update({k: torch.empty_like(gate) for k in ("out", "y", "s")})
            b[out] = b[over]
            got = forward(b)
            assert all(torch.equal(x, y) for x, y in zip(got, want)), (out, over)


@pytest.mark.parametrize("act,res", PAIRS)
@pytest.mark.parametrize("rows,dim,pad,shift", [(5, 131, 0, 0), (600, 131, 2, 3), (9, 5003, 1, 0), (4, 9001, 0, 1)])
def test_what_lies_around_the_rows_takes_no_part(L, act, res, rows, dim, pad, shift):
    """NaN between and around the rows of every input, which share vectors with the rows' ends."""
    import torch
    g = gen(31)

    def holed(dtype, mul):
        view, full = wide(rows, dim, pad, dtype, g, fill=float("nan"), shift=shift)
        view.copy_(rand((rows, dim), dtype, g, mul))
        return view
    x, h, dy, dh = holed(act, 1.0), holed(res, 2.0), holed(act, 0.1), holed(res, 0.1)
    gate, w1, w2 = holed(act, 0.5), rand((dim,), act, g, 0.2, 1.0), rand((dim,), act, g, 0.2, 1.0)
    clean = [t.contiguous() for t in (x, h, dy, dh, gate)]
    got = []
    for xx, hh, yy, dd, gg in ((x, h, dy, dh, gate), clean):
        outs = [wide(rows, dim, pad, t, g, fill=5.0, shift=shift)[0] for t in (res, act, act, act, res, act)]
        d1, d2 = torch.empty_like(w1), torch.empty_like(w2)
        L.reduce_norm([xx, yy], hh, outs[0], outs[1], sum_out=outs[2], post_weight=w1, pre_weight=w2, gate=gg, gate_rows=1)
        L.reduce_norm_backward(hh, yy, dd, outs[3], outs[4], total=xx, post_weight=w1, pre_weight=w2, gate=gg, gate_rows=1,
                               post_weight_grad=d1, pre_weight_grad=d2, gate_grad=outs[5])
        got.append(outs + [d1, d2])
    (s64, h64, y64), (ms, mh, my) = forward64([clean[0], clean[2]], clean[1], w1, w2, clean[4], 1, 1.0, 1e-6, 0.0, True)
    want, mag = backward64(clean[0], clean[1], clean[2], clean[3], w1, w2, clean[4], 1, 1.0, 1e-6, 0.0, True, True)
    deep = 128 + rows // 64 + 32
    for outs in got:
        for i, (a, m, d) in enumerate(((h64, mh, 128), (y64, my, 128), (s64, ms, 2), (want["send"], mag["send"], 256),
                                       (want["res"], mag["res"], 128), (want["gate"], mag["gate"], deep),
                                       (want["w1"], mag["w1"], deep), (want["w2"], mag["w2"], deep))):
            near(outs[i], a, m, d, i)


def test_backward_of_no_rows_writes_zero_sums(L):
    import torch
    dim = 100
    none = torch.empty((0, dim), dtype=torch.float32, device="cuda")
    w = torch.ones(dim, device="cuda")
    dw1, dw2, dg = (torch.full((dim,), 3.0, device="cuda") for _ in range(3))
    L.reduce_norm_backward(none, none, none, none, none, total=none, post_weight=w, pre_weight=w, gate=w,
                           post_weight_grad=dw1, pre_weight_grad=dw2, gate_grad=dg)
    for t in (dw1, dw2, dg):
        assert bool((t == 0).all())
    L.reduce_norm([none], none, none, none, pre_weight=w)


def test_gradients_against_differences(L):
    """d/dt of <forward(x + t v), c> at 0 by central differences of the fp32 forward pass, against <gradient, v>.  With
    t = 2^-5 the third derivative leaves about t^2 / 6 of the value's own size, the fp32 results 2^-22 of |f| / t per
    element, averaged over thousands: both far below 1 % of the derivative."""
    import torch
    g = gen(9)
    rows, dim, gate_rows = 24, 200, 5
    x = dict(a=rand((rows, dim), F32, g), b=rand((rows, dim), F32, g), res=rand((rows, dim), F32, g),
             w1=rand((dim,), F32, g, 0.1, 1.0), w2=rand((dim,), F32, g, 0.1, 1.0), gate=rand((5, dim), F32, g, 0.3, 1.0))
    ch, cy = rand((rows, dim), F32, g), rand((rows, dim), F32, g)

    def run(x):
        h, y, s = (torch.empty((rows, dim), device="cuda") for _ in range(3))
        L.reduce_norm([x["a"], x["b"]], x["res"], h, y, sum_out=s, post_weight=x["w1"], pre_weight=x["w2"], gate=x["gate"],
                      gate_rows=gate_rows, scale=0.6)
        return h, y, s

    h, y, s = run(x)
    grad = {k: torch.empty_like(v) for k, v in x.items()}
    L.reduce_norm_backward(h, cy, ch, grad["a"], grad["res"], total=s, post_weight=x["w1"], pre_weight=x["w2"],
                           gate=x["gate"], gate_rows=gate_rows, post_weight_grad=grad["w1"], pre_weight_grad=grad["w2"],
                           gate_grad=grad["gate"], scale=0.6)
    grad["b"] = grad["a"]
    for k in x:
        v = grad[k] / grad[k].double().square().mean().sqrt().float()  # along the gradient: no cancellation
        t = 2.0 ** -5
        f = []
        for sign in (1.0, -1.0):
            h, y, _ = run({**x, k: x[k] + sign * t * v})
            f.append((h.double() * ch).sum() + (y.double() * cy).sum())
        slope, want = float((f[0] - f[1]) / (2 * t)), float((grad[k].double() * v).sum())
        assert abs(slope - want) <= 0.01 * abs(want), (k, slope, want)


# ---------------------------------------------------------------- embedding

TYPES = [(BF, BF), (F16, F16), (F32, F32), (F32, BF), (F32, F16), (BF, F32), (F16, F32)]


def lookup64(table, ids, first, scale):
    import torch
    row = ids.long() - first
    here = (row >= 0) & (row < table.shape[0])
    out = torch.zeros((ids.numel(), table.shape[1]), dtype=torch.float64, device="cuda")
    out[here] = table[row[here]].double() * scale
    return out


@pytest.mark.parametrize("table_type,out_type", TYPES)
@pytest.mark.parametrize("tokens,vocab,dim,pad,shift", [(1, 1, 1, 0, 0), (7, 5, 3, 0, 0), (33, 100, 64, 0, 0),
                                                       (257, 1003, 501, 0, 1), (64, 300, 520, 8, 0), (5, 40, 8192, 0, 0),
                                                       (3, 9, 20001, 3, 0), (1000, 50, 128, 0, 0)])
def test_embedding(L, table_type, out_type, tokens, vocab, dim, pad, shift):
    import torch
    g = gen(tokens + dim)
    first = 1000
    table = wide(vocab, dim, pad, table_type, g, shift=shift)[0]
    out, full = wide(tokens, dim, pad, out_type, g, fill=5.0, shift=shift)
    ids = torch.randint(first - vocab // 2 - 1, first + vocab + vocab // 2 + 1, (tokens,), device="cuda", generator=g)
    for idt in (torch.int64, torch.int32):
        for scale in (1.0, 3.7):
            L.embedding(table, ids.to(idt), out, first=first, scale=scale)
            want = lookup64(table, ids, first, scale)
            near(out, want, want.abs(), 1, "rows")
            view = out.clone()
            out.fill_(5.0)
            assert bool((full == 5.0).all())
            assert bool((view[want.abs().sum(1) == 0] == 0).all())


def test_embedding_extreme_ids_and_nan_rows(L):
    import torch
    table = torch.randn(4, 32, device="cuda")
    table[0] = float("nan")
    big = 2 ** 63 - 1
    ids = torch.tensor([big, -big - 1, 0, -1, 4, 3, 2 ** 31, 2 ** 32 + 1, -2 ** 32 + 2], device="cuda")
    out = torch.full((9, 32), 5.0, device="cuda")
    L.embedding(table, ids, out)
    assert bool(out[2].isnan().all()) and torch.equal(out[5], table[3])
    for r in (0, 1, 3, 4, 6, 7, 8):
        assert bool((out[r] == 0).all()), r
    L.embedding(table[1:], ids, out, first=big - 1)  # ids first .. first + 2 run past the largest id
    assert torch.equal(out[0], table[2]) and bool((out[1:] == 0).all())
    L.embedding(table[1:], ids, out, first=-big - 1)
    assert torch.equal(out[1], table[1]) and bool((out[0] == 0).all()) and bool((out[2:] == 0).all())
    L.embedding(table[:0], ids, out)
    assert bool((out == 0).all())


def grad64(out_grad, ids, vocab, first, scale, old):
    import torch
    row = ids.long() - first
    here = (row >= 0) & (row < vocab)
    total = torch.zeros((vocab, out_grad.shape[1]), dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(total)
    total.index_put_((row[here],), out_grad[here].double() * scale, accumulate=True)
    mag.index_put_((row[here],), out_grad[here].double().abs() * abs(scale), accumulate=True)
    if old is not None:
        total, mag = total + old.double(), mag + old.double().abs()
    return total, mag


def some_ids(kind, tokens, vocab, first, g):
    import torch
    if kind == "same":
        return torch.full((tokens,), first + vocab // 2, device="cuda")
    if kind == "outside":
        return torch.full((tokens,), first + vocab, device="cuda")
    if kind == "distinct":
        return first + torch.randperm(max(vocab, tokens), device="cuda", generator=g)[:tokens]
    if kind == "falling":  # as words do, with a third of padding
        u = torch.rand(tokens, dtype=torch.float64, device="cuda", generator=g)
        ids = first + ((vocab * 2 + 1.0) ** u - 1.0).long()
        return torch.where(torch.rand(tokens, device="cuda", generator=g) < 0.33, first, ids)
    return torch.randint(first - vocab // 2 - 1, first + vocab + vocab // 2 + 1, (tokens,), device="cuda", generator=g)


def sum_depth(tokens):
    """A chunk of 8 to 32 tokens; then up to 64 chunks one after another, or a sixteenth of a longer row's and the
    sixteen wavefronts; a few operations at the end."""
    return 32 + max(64, tokens / 8 / 16 + 16) + 8


@pytest.mark.parametrize("table_type,out_type", TYPES)
@pytest.mark.parametrize("kind,tokens,vocab,dim,pad,shift", [
    ("random", 1, 1, 1, 0, 0), ("random", 5, 9, 3, 0, 0), ("same", 63, 7, 64, 0, 0), ("outside", 40, 7, 64, 0, 0),
    ("falling", 257, 5003, 501, 0, 0), ("falling", 3000, 300, 520, 8, 0), ("same", 5000, 3, 260, 0, 0),
    ("distinct", 2049, 3000, 96, 0, 1), ("random", 7000, 70000, 40, 0, 0), ("falling", 1500, 200, 4096, 0, 0),
    ("random", 100, 70, 20001, 3, 0)])
def test_embedding_grad(L, table_type, out_type, kind, tokens, vocab, dim, pad, shift):
    import torch
    g = gen(tokens * 7 + dim)
    first = 500
    ids = some_ids(kind, tokens, vocab, first, g)
    out_grad = wide(tokens, dim, pad, out_type, g, 0.1, shift=shift)[0]
    depth = sum_depth(tokens)
    for accumulate in (False, True):
        for idt in (torch.int64, torch.int32):
            table, full = wide(vocab, dim, pad, table_type, g, fill=5.0, shift=shift)
            old = None
            if accumulate:
                old = rand((vocab, dim), table_type, g)
                table.copy_(old)
            L.embedding_grad(out_grad, ids.to(idt), table, first=first, scale=1.5, accumulate=accumulate)
            want, mag = grad64(out_grad, ids, vocab, first, 1.5, old)
            near(table, want, mag, depth, "table")
            again = old.clone() if accumulate else torch.full_like(old if old is not None else table, 9.0)
            L.embedding_grad(out_grad, ids.to(idt), again, first=first, scale=1.5, accumulate=accumulate)
            assert torch.equal(again, table)
            if accumulate:  # rows that no id names keep their bits
                named = torch.zeros(vocab, dtype=torch.bool, device="cuda")
                row = ids - first
                named[row[(row >= 0) & (row < vocab)]] = True
                assert torch.equal(table[~named], old[~named])
            table.fill_(5.0)
            assert bool((full == 5.0).all())


def test_embedding_grad_keeps_the_order_of_tokens(L):
    """The sum runs over an id's tokens in their order: 1 + 2^-24 + ... in fp32 shows any other."""
    import torch
    tokens = 8  # one chunk
    ids = torch.tensor([3, 1, 3, 1, 3, 1, 3, 3], device="cuda")
    x = torch.tensor([1.0, 2.0 ** -24, 2.0 ** -24, 1.0, 2.0 ** -24, 2.0 ** -24, 2.0 ** -24, -1.0], device="cuda")
    grad = x[:, None].expand(tokens, 5).contiguous()
    table = torch.empty(4, 5, device="cuda")
    L.embedding_grad(grad, ids, table)
    import numpy as np
    for v in (1, 3):
        s = np.float32(0.0)
        for t in range(tokens):
            if int(ids[t]) == v:
                s = np.float32(s + np.float32(float(x[t])))
        assert float(table[v, 0]) == float(s) and torch.equal(table[v], table[v, :1].expand(5))


@pytest.mark.parametrize("dim", [5, 300])
@pytest.mark.parametrize("counts", [
    [16], [17], [15, 2], [256], [1, 255], [255, 1], [16, 16, 16], [8, 40, 3, 64, 1, 0, 33, 107], [1] * 256, [129, 128], [512], [519], [520], [521], [528], [529], [3, 513, 520, 8, 512, 1000, 1, 528, 2053], [504, 512, 8, 520, 600, 0, 1],
    [8, 505, 512, 520, 7, 1], [1, 4096], [4096, 1], [511, 1025, 16, 2, 513]], ids=lambda c: "-".join(map(str, c)))
def test_embedding_grad_rows_of_many_chunks(L, dim, counts):
    """Ids that occur about as often as 64 chunks of eight tokens hold, at every kind of place among the chunks."""
    import torch
    g = gen(sum(counts) + dim)  # up to 256 tokens: chunks of 16 in one workgroup
    tokens = sum(counts)
    ids = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), torch.tensor(counts, device="cuda"))
    ids = ids[torch.randperm(tokens, device="cuda", generator=g)]
    grad = rand((tokens, dim), F32, g)
    old = rand((len(counts), dim), F32, g)
    for accumulate in (False, True):
        table = old.clone()
        L.embedding_grad(grad, ids, table, accumulate=accumulate)
        want, mag = grad64(grad, ids, len(counts), 0, 1.0, old if accumulate else None)
        near(table, want, mag, sum_depth(tokens), "table")


@pytest.mark.parametrize("tokens,vocab", [(255, 100), (256, 2 << 20), (257, 100), (2048, 2047), (2049, 2047), (2049, 2048), (4097, 1), (30000, 3 << 20), (70000, 5), (530000, 2047)])
def test_embedding_grad_sorts(L, tokens, vocab):
    """One and several workgroups, one to two passes, tiles of one and several rounds; small whole numbers sum exactly."""
    import torch
    g = gen(tokens + vocab)
    ids = some_ids("random", tokens, vocab, 3, g)
    grad = torch.randint(-8, 9, (tokens, 2), device="cuda", generator=g).float()
    table = torch.full((vocab, 2), 9.0, device="cuda")
    L.embedding_grad(grad, ids, table, first=3)
    want, _ = grad64(grad, ids, vocab, 3, 1.0, None)
    assert torch.equal(table.double(), want)


def test_embedding_grad_without_tokens(L):
    import torch
    ids = torch.empty(0, dtype=torch.int64, device="cuda")
    grad = torch.empty(0, 16, device="cuda")
    table = torch.full((5, 16), 3.0, device="cuda")
    L.embedding_grad(grad, ids, table, accumulate=True)
    assert bool((table == 3).all())
    L.embedding_grad(grad, ids, table)
    assert bool((table == 0).all())
    L.embedding(table, ids, grad)


@pytest.mark.parametrize("tokens", [200, 600, 5000])
def test_embedding_grad_nan_stays_in_its_row(L, tokens):
    """Neither a token's NaN nor that of a token of another shard reaches a row that does not name it."""
    import torch
    g = gen(11)
    grad = rand((tokens, 70), F32, g)
    ids = torch.randint(0, 30, (tokens,), device="cuda", generator=g)
    a, b = torch.empty(20, 70, device="cuda"), torch.empty(20, 70, device="cuda")
    L.embedding_grad(grad, ids, a)
    one = int((ids < 20).nonzero()[7])
    grad[one] = float("nan")
    grad[ids >= 20] = float("inf")
    L.embedding_grad(grad, ids, b)
    hit = int(ids[one])
    for v in range(20):
        assert bool(b[v].isnan().all()) if v == hit else torch.equal(a[v], b[v])


def test_scales_of_every_kind(L):
    """Rows that the shard does not have are +0 whatever the scale, others what the formula says."""
    import torch
    table = torch.randn(4, 40, device="cuda")
    ids = torch.tensor([1, 7, 3, -2], device="cuda")
    for scale in (-2.0, 0.0, float("inf"), float("nan"), 1e-30):
        out = torch.full((4, 40), 5.0, device="cuda")
        L.embedding(table, ids, out, scale=scale)
        assert bool((out[[1, 3]].view(torch.int32) == 0).all())
        want = table[[1, 3]] * torch.tensor(scale, device="cuda")
        assert torch.equal(out[[0, 2]].nan_to_num(7.0), want.nan_to_num(7.0))
        for tokens in (4, 1200):
            many = ids.repeat(tokens // 4)
            grad = torch.ones(tokens, 40, device="cuda")
            t = torch.full((4, 40), 5.0, device="cuda")
            L.embedding_grad(grad, many, t, scale=scale)
            assert bool((t[[0, 2]].view(torch.int32) == 0).all())
            want = torch.full((2, 40), tokens / 4, device="cuda") * torch.tensor(scale, device="cuda")
            assert torch.equal(t[[1, 3]].nan_to_num(7.0), want.nan_to_num(7.0))


# --------------------------------------------------- offsets, streams, graphs

def test_offsets_beyond_32_bits(L):
    """Rows of one matrix more than 4 GiB apart, a table of more than 4 GiB."""
    import torch
    if torch.cuda.get_device_properties(0).total_memory < 64 << 30:
        pytest.skip("needs memory")
    g = gen(12)
    dim, stride = 264, (1 << 31) + 8
    pool = torch.empty(2 * stride + dim, dtype=torch.bfloat16, device="cuda")
    far = pool.as_strided((3, dim), (stride, 1))
    src, w = rand((3, dim), BF, g), rand((dim,), BF, g, 0.1, 1.0)
    far.copy_(rand((3, dim), BF, g))
    before = far.clone()
    y, s = torch.empty_like(src), torch.empty_like(src)
    L.reduce_norm([src], far, far, y, sum_out=s, post_weight=w, pre_weight=w)
    (_, wh, wy), (_, mh, my) = forward64([src], before, w, w, None, 0, 1.0, 1e-6, 0.0, True)
    near(far, wh, mh, 128, "stream")
    near(y, wy, my, 128, "norm")
    dres = torch.empty_like(src)
    L.reduce_norm_backward(far, y, src, None, dres, total=s, post_weight=w, pre_weight=w)
    want, mag = backward64(s, far, y, src, w, w, None, 0, 1.0, 1e-6, 0.0, True, True)
    near(dres, want["res"], mag["res"], 128, "res")
    del pool, far
    vocab, dim = 70000, 32776
    table = torch.empty((vocab, dim), dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([69999, 65536, 3, 70000, 69999], device="cuda")
    grad = rand((5, dim), BF, g)
    table.fill_(1.0)
    L.embedding_grad(grad, ids, table)
    want = torch.stack([grad[2].double(), grad[1].double(), grad[0].double() + grad[4].double()])
    near(table[[3, 65536, 69999]], want, want.abs(), 4, "table")
    assert int((table != 0).any(1).sum()) == 3
    out = torch.empty((5, dim), dtype=torch.bfloat16, device="cuda")
    L.embedding(table, ids, out)
    assert torch.equal(out[0], table[69999]) and torch.equal(out[1], table[65536]) and bool((out[3] == 0).all())


def test_more_rows_than_workgroups(L):
    """Some rows are a workgroup's second ones (a million workgroups of four rows, of eight tokens)."""
    import torch
    g = gen(21)
    rows, dim = (4 << 20) + 4099, 8
    src, res = rand((rows, dim), BF, g), rand((rows, dim), BF, g)
    h, y, s = torch.empty_like(res), torch.empty_like(res), torch.empty_like(res)
    L.reduce_norm([src, res], res, h, y, sum_out=s, post_norm=True)
    (ws, wh, wy), (ms, mh, my) = forward64([src, res], res, None, None, None, 0, 1.0, 1e-6, 0.0, True)
    near(h, wh, mh, 128, "stream")
    near(y, wy, my, 128, "norm")
    near(s, ws, ms, 1, "sum")
    del src, res, h, y, s, ws, wh, wy, ms, mh, my
    tokens = (8 << 20) + 4097
    table = rand((1000, 3), F32, g)
    ids = torch.randint(-10, 1010, (tokens,), device="cuda", generator=g)
    for width in (1, 3):
        out = torch.full((tokens, width), 5.0, device="cuda")
        L.embedding(table[:, :width], ids, out)
        here = (ids >= 0) & (ids < 1000)
        assert torch.equal(out[here], table[:, :width][ids[here]]) and bool((out[~here] == 0).all())


def test_one_group_of_gates_however_long(L):
    import torch
    g = gen(22)
    rows, dim = 37, 640
    src, res, dy, dh = (rand((rows, dim), BF, g) for _ in range(4))
    gate = rand((1, dim), BF, g)
    got = []
    for gate_rows in (0, rows, rows + 1, 1 << 40, (1 << 63) - 1):
        h, y, s, ds, dg = (torch.empty_like(t) for t in (res, res, res, res, gate))
        L.reduce_norm([src], res, h, y, sum_out=s, gate=gate, gate_rows=gate_rows)
        L.reduce_norm_backward(h, dy, dh, ds, total=s, gate=gate, gate_rows=gate_rows, gate_grad=dg)
        got.append((h, y, ds, dg))
        assert all(torch.equal(a, b) for a, b in zip(got[0], got[-1])), gate_rows
    want, mag = backward64(s, h, dy, dh, None, None, gate, 0, 1.0, 1e-6, 0.0, False, True)
    near(dg[0], want["gate"], mag["gate"], 128 + 4 + 32, "gate")


def test_other_streams_and_their_workspaces(L):
    import torch
    g = gen(13)
    grad, ids = rand((3000, 128), BF, g), torch.randint(0, 500, (3000,), device="cuda", generator=g)
    x, h = rand((2000, 256), BF, g), rand((2000, 256), BF, g)
    w = rand((256,), BF, g, 0.1, 1.0)
    want_t, want_d, want_w = torch.empty(500, 128, device="cuda"), torch.empty_like(x), torch.empty_like(w)
    L.embedding_grad(grad, ids, want_t)
    L.reduce_norm_backward(h, x, h, want_d, total=x, post_weight=w, pre_weight=w, post_weight_grad=want_w)
    torch.cuda.synchronize()
    with pytest.raises(L.FlagcxError):  # memory of the current stream is not for another one
        L.embedding_grad(grad, ids, want_t, stream=L.Stream(torch.cuda.Stream().cuda_stream))
    runs = []
    for k in range(3):
        st = torch.cuda.Stream()
        ws = torch.empty(L.embedding_grad_workspace(3000, 500, 128), dtype=torch.uint8, device="cuda")
        ws2 = torch.empty(L.reduce_norm_backward_workspace(2000, 256), dtype=torch.uint8, device="cuda")
        runs.append((st, ws, ws2, torch.empty_like(want_t), torch.empty_like(want_d), torch.empty_like(want_w)))
    torch.cuda.synchronize()
    for st, ws, ws2, t, d, dw in runs:  # at the same time, each with its own workspace
        L.embedding_grad(grad, ids, t, workspace=ws, stream=L.Stream(st.cuda_stream))
        L.reduce_norm_backward(h, x, h, d, total=x, post_weight=w, pre_weight=w, post_weight_grad=dw, workspace=ws2,
                               stream=L.Stream(st.cuda_stream))
    torch.cuda.synchronize()
    for _, _, _, t, d, dw in runs:
        assert torch.equal(t, want_t) and torch.equal(d, want_d) and torch.equal(dw, want_w)
    t = torch.empty_like(want_t)
    L.embedding_grad(grad, ids, t, workspace=runs[0][1], stream=None)  # the NULL stream: done when the call returns
    assert torch.equal(t, want_t)
    short = torch.empty(L.embedding_grad_workspace(3000, 500, 128) - 1, dtype=torch.uint8, device="cuda")
    with pytest.raises(L.FlagcxError):
        L.embedding_grad(grad, ids, t, workspace=short)


def test_refusals_of_the_binding(L):
    import torch
    x = torch.zeros(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    wrong = [
        lambda: L.reduce_norm([x, x[:, :4]], x, torch.zeros_like(x), torch.zeros_like(x)),
        lambda: L.reduce_norm([x, x.half()], x, torch.zeros_like(x), torch.zeros_like(x)),
        lambda: L.reduce_norm([x[:1].expand(4, 8)], x, torch.zeros_like(x), torch.zeros_like(x)),
        lambda: L.reduce_norm([x.t().contiguous().t()], x, torch.zeros_like(x), torch.zeros_like(x)),
        lambda: L.reduce_norm([x, torch.zeros(4, 16, device="cuda")[:, :8]], x, torch.zeros_like(x), torch.zeros_like(x)),
        lambda: L.reduce_norm([x], x, torch.zeros_like(x), torch.zeros_like(x), post_weight=w, pre_weight=w.half()),
        lambda: L.reduce_norm([x], x, torch.zeros_like(x), torch.zeros_like(x), gate=w[:4]),
        lambda: L.reduce_norm([x], x, torch.zeros_like(x), torch.zeros_like(x), gate=x, gate_rows=2),
        lambda: L.reduce_norm([x], x, torch.zeros_like(x), torch.zeros_like(x), gate=x, gate_rows=-1),
        lambda: L.reduce_norm([x], x.cpu(), torch.zeros_like(x), torch.zeros_like(x)),
        lambda: L.reduce_norm([x.double()], x, torch.zeros_like(x), torch.zeros_like(x)),
        lambda: L.reduce_norm([x.int()], x.int(), torch.zeros_like(x).int()),
        lambda: L.embedding(x, ids.short(), torch.zeros_like(x)),
        lambda: L.embedding(x, ids[::2], torch.zeros(2, 8, device="cuda")),
        lambda: L.embedding(x, ids, torch.zeros(3, 8, device="cuda")),
        lambda: L.embedding(x.bfloat16(), ids, torch.zeros(4, 8, device="cuda", dtype=torch.float16)),
        lambda: L.embedding_grad(x, ids, x),
        lambda: L.embedding_grad(x[:, :4], ids, torch.zeros_like(x)),
        lambda: L.reduce_norm_backward(x, x, x, torch.zeros_like(x), total=None, post_weight=w),
    ]
    for k, call in enumerate(wrong):
        with pytest.raises(L.FlagcxError) as e:
            call()
        assert e.value.code == int(L.Result.InvalidArgument), k


def test_captured_calls_replay(L):
    """All four calls captured into one graph, replayed on new inputs with eager calls in between; a second graph with
    workspaces of its own replays next to it."""
    import torch
    g = gen(14)
    tokens, vocab, dim = 3000, 700, 384
    ids = torch.randint(0, vocab, (tokens,), device="cuda", generator=g)
    table = rand((vocab, dim), F32, g)
    w = rand((dim,), F32, g, 0.1, 1.0)
    gate = rand((3, dim), BF, g, 0.3, 0.5)

    def make():
        e = lambda d: torch.empty((tokens, dim), dtype=dt(d), device="cuda")
        return dict(x=e(BF), h=e(F32), y=e(BF), s=e(BF), ds=e(BF), dres=e(F32), dw=torch.empty_like(w),
                    dg=torch.empty_like(gate), dt=torch.empty_like(table), ws=torch.empty(
                        L.embedding_grad_workspace(tokens, vocab, dim), dtype=torch.uint8, device="cuda"),
                    ws2=torch.empty(L.reduce_norm_backward_workspace(tokens, dim, True, 1024), dtype=torch.uint8, device="cuda"))

    def run(b):
        L.embedding(table, ids, b["x"], scale=2.0)
        L.reduce_norm([b["x"], b["x"]], None, b["h"], b["y"], sum_out=b["s"], post_weight=w, pre_weight=w, gate=gate,
                      gate_rows=1024)
        L.reduce_norm_backward(b["h"], b["y"], b["h"], b["ds"], b["dres"], total=b["s"], post_weight=w, pre_weight=w,
                               gate=gate, gate_rows=1024, post_weight_grad=b["dw"], gate_grad=b["dg"], workspace=b["ws2"])
        L.embedding_grad(b["ds"], ids, b["dt"], scale=2.0, workspace=b["ws"])

    eager, a, b = make(), make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for buf in (a, b):
        with torch.cuda.stream(side):
            run(buf)
        side.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side, capture_error_mode="global"):
            run(buf)
        graphs.append(gr)
    other = torch.cuda.Stream()
    for rep in range(4):
        ids.copy_(torch.randint(-50, vocab + 50, (tokens,), device="cuda", generator=g))
        table.copy_(rand((vocab, dim), F32, g))
        for buf in (a, b):
            for k in ("h", "y", "s", "ds", "dres", "dw", "dg", "dt"):
                buf[k].fill_(7.0)
            buf["ws"].fill_(rep)
            buf["ws2"].fill_(rep)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        run(eager)
        torch.cuda.synchronize()
        for k in ("x", "h", "y", "s", "ds", "dres", "dw", "dg", "dt"):
            assert torch.equal(a[k], eager[k]), (rep, k)
            assert torch.equal(b[k], eager[k]), (rep, k)


# ---------------------------------------------------------- as they are used

@pytest.mark.parametrize("act,res", [(F32, F32), (BF, F32), (BF, BF)])
def test_a_training_step_of_a_tensor_parallel_model(L, act, res):
    """Two ranks on one GPU: the shards' lookups are folded, two blocks end in reduce_norm (partial results: a product
    of the normed stream with each rank's share of the weights, columnwise), and the gradients go back into each rank's
    shard.  Against the same model in 64-bit autograd; with 16-bit values in between, every tensor that is stored is off
    by 2^-9 of its size at most once on the way, about ten of them in a chain: 5 % of the gradient's norm is far above
    that and far below any wrong term."""
    import torch
    g = gen(15)
    tokens, vocab, dim, ranks, eps = 60, 40, 96, 2, 1e-5
    shard = vocab // ranks
    tables = [rand((shard, dim), res, g) for _ in range(ranks)]
    ids = torch.randint(0, vocab, (tokens,), device="cuda", generator=g)
    mix = [[rand((dim,), act, g, 0.5, 0.3) for _ in range(ranks)] for _ in range(2)]
    pre = [rand((dim,), F32, g, 0.1, 1.0) for _ in range(3)]
    post = [rand((dim,), F32, g, 0.1, 1.0) for _ in range(2)]
    gates = [rand((3, dim), act, g, 0.3, 0.7) for _ in range(2)]
    target = rand((tokens, dim), act, g)
    e = lambda d: torch.empty((tokens, dim), dtype=dt(d), device="cuda")

    # forward: the entrance's fold is a block end without a residual
    parts = [L.embedding(tables[r], ids, e(act), first=r * shard, scale=dim ** 0.5) for r in range(ranks)]
    h, y = [e(res)], [e(act)]
    L.reduce_norm(parts, None, h[0], y[0], pre_weight=pre[0], eps=eps)
    sums = []
    for b in range(2):
        part = [(y[b].float() * mix[b][r].float()).to(dt(act)) for r in range(ranks)]
        h.append(e(res)), y.append(e(act)), sums.append(e(act))
        L.reduce_norm(part, h[b], h[b + 1], y[b + 1], sum_out=sums[b], post_weight=post[b], pre_weight=pre[b + 1],
                      gate=gates[b], gate_rows=20, scale=0.8, eps=eps)
    # backward of sum(y * target) / 8
    dy, dh = (target.float() / 8).to(dt(act)), None
    got = {}
    for b in (1, 0):
        ds, dres = e(act), e(res)
        dpost, dpre, dgate = torch.empty_like(post[b]), torch.empty_like(pre[b + 1]), torch.empty_like(gates[b])
        L.reduce_norm_backward(h[b + 1], dy, dh, ds, dres, total=sums[b], post_weight=post[b], pre_weight=pre[b + 1],
                               gate=gates[b], gate_rows=20, post_weight_grad=dpost, pre_weight_grad=dpre,
                               gate_grad=dgate, scale=0.8, eps=eps)
        got.update({("post", b): dpost, ("pre", b + 1): dpre, ("gate", b): dgate})
        dys = [(ds.float() * mix[b][r].float()).to(dt(act)) for r in range(ranks)]
        dy, dh = e(act), dres
        L.reduce(dys, dy, L.RedOp.Sum)
    ds, dpre = e(act), torch.empty_like(pre[0])
    L.reduce_norm_backward(h[0], dy, dh, ds, pre_weight=pre[0], pre_weight_grad=dpre, eps=eps)
    got["pre", 0] = dpre
    for r in range(ranks):
        got["table", r] = L.embedding_grad(ds, ids, torch.empty_like(tables[r]), first=r * shard, scale=dim ** 0.5)

    # the same in 64 bits
    leaf = lambda t: t.double().requires_grad_()
    T, P, Q, G = [leaf(t) for t in tables], [leaf(t) for t in pre], [leaf(t) for t in post], [leaf(t) for t in gates]
    norm = lambda x, w: x * (x.square().mean(1, keepdim=True) + eps) ** -0.5 * w
    x = torch.cat(T)[ids] * dim ** 0.5
    z = norm(x, P[0])
    for b in range(2):
        u = norm(sum(z * mix[b][r].double() for r in range(ranks)), Q[b])
        x = x + 0.8 * u * G[b].repeat_interleave(20, 0)
        z = norm(x, P[b + 1])
    (z * target.double() / 8).sum().backward()
    allowed = 1e-4 if act == F32 else 0.05
    for key, value in got.items():
        want = {"post": Q, "pre": P, "gate": G, "table": T}[key[0]][key[1]].grad
        rel = float((value.double() - want).norm() / want.norm())
        assert rel <= allowed, (key, rel)
