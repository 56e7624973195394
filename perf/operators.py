"""The operators around the folds of a tensor-parallel model's residual stream, as they are measured.

Four operators, two of them the gradients of the other two:

  norm       fold of the ranks' partial results, norm after the block, gate, residual scale, residual add, norm before
             the next block
  norm_grad  its gradients
  embed      rows of a table (or of one rank's shard of it) by token id, scaled; a row of zeros where another rank has it
  embed_grad the table's gradient, summed over the tokens that hold an id

`run` computes them in elementary torch operations, or through flagcx_amd.local where `own` is true.
"""
import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


# ------------------------------------------------------------------ cases

def _norm(name, ranks, rows, dim, dtype, residual, **more):
    case = {"name": name, "op": "norm", "ranks": ranks, "rows": rows, "dim": dim, "dtype": dtype, "residual": residual,
            "weight": dtype, "post": False, "gate": "none", "gate_rows": 0, "scale": 1.0, "offset": 0.0, "keep_sum": False,
            "pad": 0}
    case.update(more)
    return case


def _norm_grad(name, rows, dim, dtype, residual, **more):
    case = {"name": name, "op": "norm_grad", "rows": rows, "dim": dim, "dtype": dtype, "residual": residual, "weight": dtype,
            "post": True, "gate": "none", "gate_rows": 0, "scale": 1.0, "offset": 0.0, "pad": 0}
    case.update(more)
    return case


def _embed(name, tokens, vocab, shard, first, dim, table, dtype, **more):
    case = {"name": name, "op": "embed", "tokens": tokens, "vocab": vocab, "shard": shard, "first": first, "dim": dim,
            "table": table, "dtype": dtype, "scale": 1.0, "wide": True, "pad_share": 0.0}
    case.update(more)
    return case


def _embed_grad(name, tokens, vocab, shard, first, dim, table, dtype, **more):
    case = _embed(name, tokens, vocab, shard, first, dim, table, dtype, accumulate=False)
    case["op"] = "embed_grad"
    case.update(more)
    return case


def listed():
    return [
        # one decoding step of eight sequences over eight tensor-parallel ranks: the call is all latency
        _norm("block end, decoding", 8, 8, 8192, "bf16", "bf16"),
        # the prompt of a model with norms on both sides of every block and a residual stream in fp32
        _norm("block end, prompt", 4, 8192, 4096, "bf16", "fp32", post=True, scale=0.5, offset=1.0),
        # a training step's forward pass, gates made from each sequence's conditioning, the sum kept for the backward pass
        _norm("block end, training", 2, 16384, 6144, "bf16", "fp32", post=True, gate="rows", gate_rows=2048, keep_sum=True,
              weight="fp32"),
        # a ragged batch of an odd width, rows inside wider ones, a learned gate for each channel
        _norm("block end, odd rows", 3, 1001, 2047, "fp16", "fp16", post=True, gate="vector", weight="fp32", pad=2),
        # the same training step's backward pass
        _norm_grad("block end gradient, training", 16384, 6144, "bf16", "fp32", gate="rows", gate_rows=2048, weight="fp32"),
        # a small model trained in fp32, a gate for every token, an odd width
        _norm_grad("block end gradient, odd rows", 517, 1535, "fp32", "fp32", gate="rows", gate_rows=1, scale=0.7),
        # one decoding step of 32 sequences: one of eight ranks looks its shard up
        _embed("lookup, decoding shard", 32, 131072, 16384, 32768, 8192, "bf16", "bf16", scale=8192.0 ** 0.5),
        # a training batch, master weights in fp32, activations in bf16, ids in 32 bits
        _embed("lookup, training", 65536, 131072, 131072, 0, 4096, "fp32", "bf16", wide=False),
        # the whole table's gradient of a training batch, written from nothing
        _embed_grad("table gradient, dense", 32768, 131072, 131072, 0, 4096, "bf16", "bf16"),
        # one of eight ranks adds a micro batch to its shard's fp32 gradient
        _embed_grad("table gradient, accumulated shard", 65536, 131072, 16384, 0, 4096, "fp32", "bf16", accumulate=True,
                    scale=64.0, wide=False),
        # a padded batch: more than half of its tokens are the padding id
        _embed_grad("table gradient, padded batch", 16384, 32768, 32768, 0, 2048, "fp32", "fp32", pad_share=0.6),
        # a fine-tuning step on a small vocabulary of an odd size, an odd width
        _embed_grad("table gradient, small odd", 257, 5003, 5003, 0, 501, "fp16", "fp16", scale=0.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dim(rng):
    d = _log_int(rng, 64, 8192)
    return d if rng.random() < 0.3 else max(64, d // 64 * 64)


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "embed", "embed_grad"])
    dim = _dim(rng)
    if op in ("norm", "norm_grad"):
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        residual = rng.choice([dtype, "fp32"])
        ranks = rng.randint(1, 8) if op == "norm" else 1
        most = 16384 * 6144 * 3 // (dim * (ranks + 3))
        rows = _log_int(rng, 1, min(32768, max(2, most)))
        gate = rng.choice(["none", "vector", "rows"])
        common = dict(weight=rng.choice([dtype, "fp32"]), post=rng.random() < 0.6, gate=gate,
                      gate_rows=_log_int(rng, 1, rows) if gate == "rows" else 0, scale=round(rng.uniform(0.1, 1.5), 3),
                      offset=rng.choice([0.0, 1.0]), pad=rng.choice([0, 0, 0, 64, 5]))
        if op == "norm":
            case = _norm("", ranks, rows, dim, dtype, residual, keep_sum=rng.random() < 0.5, **common)
        else:
            case = _norm_grad("", rows, dim, dtype, residual, **common)
    else:
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        table = rng.choice([dtype, "fp32"])
        vocab = _log_int(rng, 500, 131072)
        parts = rng.choice([1, 1, 2, 8])
        shard = max(1, vocab // parts)
        most = min(65536, 32768 * 4096 // dim)
        common = dict(scale=round(rng.uniform(0.5, 64.0), 3), wide=rng.random() < 0.5, pad_share=rng.choice([0.0, 0.0, 0.3, 0.6]))
        args = ("", _log_int(rng, 1, most), vocab, shard, rng.randrange(parts) * shard, dim, table, dtype)
        case = _embed(*args, **common) if op == "embed" else _embed_grad(*args, accumulate=rng.random() < 0.5, **common)
    del case["name"]
    return case


# ----------------------------------------------------------------- inputs

def _gate_count(case):
    if case["gate"] == "vector":
        return 1
    return -(-case["rows"] // case["gate_rows"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, mul=1.0, add=0.0):
        x = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, 1.0, generator=gen)
        return x.mul_(mul).add_(add).to(_DT[dtype])

    def rows_of(dtype, mul):  # rows that may lie inside wider ones
        return normal((case["rows"], case["dim"] + case["pad"]), dtype, mul)[:, :case["dim"]]

    def empty(shape, dtype):
        return torch.empty(shape, dtype=_DT[dtype], device="cuda")

    s = {"case": case}
    if case["op"] in ("norm", "norm_grad"):
        rows, dim, dtype, residual = case["rows"], case["dim"], case["dtype"], case["residual"]
        near = 1.0 - case["offset"]  # weights learn around one; with an offset of one they are held around zero
        s["post_weight"] = normal((dim,), case["weight"], 0.1, near) if case["post"] else None
        s["pre_weight"] = normal((dim,), case["weight"], 0.1, near)
        s["gate"] = None
        if case["gate"] == "vector":
            s["gate"] = normal((dim,), dtype, 0.3, 0.5)
        elif case["gate"] == "rows":
            s["gate"] = normal((_gate_count(case), dim), dtype, 0.3, 0.5)
        if case["op"] == "norm":
            s["partials"] = [rows_of(dtype, case["ranks"] ** -0.5) for _ in range(case["ranks"])]
            s["stream"] = rows_of(residual, 2.0)
            s["sum_out"] = empty((rows, dim), dtype) if case["keep_sum"] else None
            s["stream_out"], s["norm_out"] = empty((rows, dim), residual), empty((rows, dim), dtype)
        else:
            s["sum"] = rows_of(dtype, 1.0)
            s["stream_out"] = rows_of(residual, 2.0)
            s["norm_grad"], s["stream_out_grad"] = rows_of(dtype, 1e-2), rows_of(residual, 1e-2)
            s["send_grad"], s["stream_grad"] = empty((rows, dim), dtype), empty((rows, dim), residual)
            s["post_weight_grad"] = empty((dim,), case["weight"]) if case["post"] else None
            s["pre_weight_grad"] = empty((dim,), case["weight"])
            s["gate_grad"] = None if s["gate"] is None else torch.empty_like(s["gate"])
        return s
    # ids fall off as words do, with the inverse of their rank; padding is the first id
    u = torch.rand(case["tokens"], dtype=torch.float64, device="cuda", generator=gen)
    ids = ((case["vocab"] + 1.0) ** u - 1.0).long().clamp_(0, case["vocab"] - 1)
    is_pad = torch.rand(case["tokens"], device="cuda", generator=gen) < case["pad_share"]
    ids = ids.masked_fill_(is_pad, 0)
    s["ids"] = ids if case["wide"] else ids.int()
    if case["op"] == "embed":
        s["table"] = normal((case["shard"], case["dim"]), case["table"], 0.02)
        s["out"] = empty((case["tokens"], case["dim"]), case["dtype"])
    else:
        s["out_grad"] = normal((case["tokens"], case["dim"]), case["dtype"], 1e-2)
        held = case["accumulate"]
        s["table_grad"] = normal((case["shard"], case["dim"]), case["table"], 1e-2) if held else \
            empty((case["shard"], case["dim"]), case["table"])
    return s


# ------------------------------------------------------------- plain forms

def _gate_of_rows(s, case):
    if s["gate"] is None:
        return None
    g = s["gate"].float()
    if case["gate"] == "vector":
        return g[None, :]
    if case["gate_rows"] == 1:
        return g
    return g[torch.arange(case["rows"], device="cuda") // case["gate_rows"]]


def _plain_norm(s, case):
    total = s["partials"][0].float()
    for p in s["partials"][1:]:
        total = total + p.float()
    u = total
    if case["post"]:
        u = u * torch.rsqrt(u.square().mean(1, keepdim=True) + EPS) * (s["post_weight"].float() + case["offset"])
    g = _gate_of_rows(s, case)
    if g is not None:
        u = u * g
    h = s["stream"].float() + u * case["scale"]
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * (s["pre_weight"].float() + case["offset"])
    out = {"stream": h.to(_DT[case["residual"]]), "norm": y.to(_DT[case["dtype"]])}
    if case["keep_sum"]:
        out["sum"] = total.to(_DT[case["dtype"]])
    return out


def _plain_norm_grad(s, case):
    dt, wt, rt = _DT[case["dtype"]], _DT[case["weight"]], _DT[case["residual"]]
    total, h, dy = s["sum"].float(), s["stream_out"].float(), s["norm_grad"].float()
    r2 = torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)
    hat = h * r2
    dyw = dy * (s["pre_weight"].float() + case["offset"])
    d = s["stream_out_grad"].float() + r2 * (dyw - hat * (dyw * hat).mean(1, keepdim=True))
    out = {"stream": d.to(rt), "pre_weight": (dy * hat).sum(0).to(wt)}
    u = total
    if case["post"]:
        r1 = torch.rsqrt(total.square().mean(1, keepdim=True) + EPS)
        sat, w1 = total * r1, s["post_weight"].float() + case["offset"]
        u = sat * w1
    g = _gate_of_rows(s, case)
    e = d * case["scale"]
    if g is not None:
        dg = e * u
        if case["gate"] == "vector":
            dg = dg.sum(0)
        elif case["gate_rows"] > 1:
            short = _gate_count(case) * case["gate_rows"] - case["rows"]
            dg = torch.cat([dg, dg.new_zeros(short, case["dim"])]).view(-1, case["gate_rows"], case["dim"]).sum(1)
        out["gate"] = dg.to(dt)
        e = e * g
    if case["post"]:
        out["post_weight"] = (e * sat).sum(0).to(wt)
        e = e * w1
        e = r1 * (e - sat * (e * sat).mean(1, keepdim=True))
    out["send"] = e.to(dt)
    return out


def _rows_in_shard(s, case):
    """The shard's row of each token; one past the last where another rank has it."""
    row = s["ids"].long() - case["first"]
    return torch.where((row >= 0) & (row < case["shard"]), row, case["shard"])


def _plain_embed(s, case):
    row = _rows_in_shard(s, case)
    here = row < case["shard"]
    x = s["table"][torch.where(here, row, 0)].float() * case["scale"]
    return (x * here[:, None]).to(_DT[case["dtype"]])


def _plain_embed_grad(s, case):
    row = _rows_in_shard(s, case)
    total = torch.zeros((case["shard"] + 1, case["dim"]), dtype=torch.float32, device="cuda")
    total.index_add_(0, row, s["out_grad"].float())
    total = total[:case["shard"]] * case["scale"]
    if case["accumulate"]:
        return s["table_grad"].copy_(s["table_grad"].float() + total)
    return total.to(_DT[case["table"]])


# ------------------------------------------------------------------- calls

def _own_norm(s, case):
    from flagcx_amd import local as L
    L.reduce_norm(s["partials"], s["stream"], s["stream_out"], s["norm_out"], sum_out=s["sum_out"],
                  post_weight=s["post_weight"], pre_weight=s["pre_weight"], gate=s["gate"], gate_rows=case["gate_rows"],
                  scale=case["scale"], eps=EPS, weight_offset=case["offset"])
    out = {"stream": s["stream_out"], "norm": s["norm_out"]}
    if case["keep_sum"]:
        out["sum"] = s["sum_out"]
    return out


def _own_norm_grad(s, case):
    from flagcx_amd import local as L
    L.reduce_norm_backward(s["stream_out"], s["norm_grad"], s["stream_out_grad"], s["send_grad"], s["stream_grad"],
                           total=s["sum"], post_weight=s["post_weight"], pre_weight=s["pre_weight"], gate=s["gate"],
                           gate_rows=case["gate_rows"], post_weight_grad=s["post_weight_grad"],
                           pre_weight_grad=s["pre_weight_grad"], gate_grad=s["gate_grad"], scale=case["scale"], eps=EPS,
                           weight_offset=case["offset"])
    out = {"stream": s["stream_grad"], "pre_weight": s["pre_weight_grad"], "send": s["send_grad"]}
    if case["post"]:
        out["post_weight"] = s["post_weight_grad"]
    if s["gate"] is not None:
        out["gate"] = s["gate_grad"]
    return out


def _own_embed(s, case):
    from flagcx_amd import local as L
    return L.embedding(s["table"], s["ids"], s["out"], first=case["first"], scale=case["scale"])


def _own_embed_grad(s, case):
    from flagcx_amd import local as L
    return L.embedding_grad(s["out_grad"], s["ids"], s["table_grad"], first=case["first"], scale=case["scale"],
                            accumulate=case["accumulate"])


def run(state):
    case = state["case"]
    if own:
        f = {"norm": _own_norm, "norm_grad": _own_norm_grad, "embed": _own_embed, "embed_grad": _own_embed_grad}
    else:
        f = {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "embed": _plain_embed, "embed_grad": _plain_embed_grad}
    return f[case["op"]](state, case)


# -------------------------------------------------------------------- work

def _distinct(case):
    """Expected (distinct rows of the shard that the batch names, tokens that name one)."""
    at = np.arange(case["shard"], dtype=np.float64) + case["first"]
    p = np.log((at + 2.0) / (at + 1.0)) / math.log(case["vocab"] + 1.0) * (1.0 - case["pad_share"])
    if case["first"] == 0:
        p[0] += case["pad_share"]
    p = np.minimum(p, 1.0)
    with np.errstate(divide="ignore"):
        return float(-np.expm1(case["tokens"] * np.log1p(-p)).sum()), float(case["tokens"] * p.sum())


def work(case):
    d, dim = _SIZE[case["dtype"]], case["dim"]
    if case["op"] in ("norm", "norm_grad"):
        r, w, n = _SIZE[case["residual"]], _SIZE[case["weight"]], case["rows"] * case["dim"]
        norms = 2 if case["post"] else 1
        gates = 0 if case["gate"] == "none" else _gate_count(case) * dim * d
        if case["op"] == "norm":
            moved = n * (case["ranks"] * d + 2 * r + d + (d if case["keep_sum"] else 0)) + norms * dim * w + gates
            return {"bytes": moved, "flops": n * (case["ranks"] - 1 + 5 * norms + 4)}
        reads_sum = case["post"] or case["gate"] != "none"
        return {"bytes": n * (3 * r + 2 * d + (d if reads_sum else 0)) + 2 * norms * dim * w + 2 * gates,
                "flops": n * (11 * norms + 6)}
    t, ids = _SIZE[case["table"]], case["tokens"] * (8 if case["wide"] else 4)
    rows, named = _distinct(case)
    if case["op"] == "embed":
        return {"bytes": rows * dim * t + case["tokens"] * dim * d + ids, "flops": named * dim}
    written = 2 * rows * dim * t if case["accumulate"] else case["shard"] * dim * t
    return {"bytes": named * dim * d + written + ids, "flops": named * dim + rows * dim}


# ------------------------------------------------------------------- exact

def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)

    def f64(t):
        return None if t is None else t.to(torch.float64)

    if case["op"] in ("norm", "norm_grad"):
        dim, o, scale = case["dim"], case["offset"], case["scale"]
        w1, w2 = f64(s["post_weight"]), f64(s["pre_weight"])
        g = f64(s["gate"])
        if g is not None:
            g = g.reshape(-1, dim)
            each = case["rows"] if case["gate"] == "vector" else case["gate_rows"]
            g = g.repeat_interleave(each, 0)[:case["rows"]]

    if case["op"] == "norm":
        total = torch.zeros((case["rows"], dim), dtype=torch.float64, device="cuda")
        for p in s["partials"]:
            total += p
        u = total.clone()
        if w1 is not None:
            u *= (w1 + o) / ((total * total).sum(1, keepdim=True) / dim + EPS).sqrt()
        if g is not None:
            u *= g
        h = f64(s["stream"]) + scale * u
        out = {"stream": h, "norm": h / ((h * h).sum(1, keepdim=True) / dim + EPS).sqrt() * (w2 + o)}
        if case["keep_sum"]:
            out["sum"] = total
        return out

    if case["op"] == "norm_grad":
        # d/dx of x_i w_i (m + eps)^-1/2 with m = sum x^2 / dim, contracted with c:
        #   c_i w_i q - x_i q^3 / dim * sum_j c_j w_j x_j,  q = (m + eps)^-1/2
        def back(x, w, c):
            q = 1.0 / ((x * x).sum(1, keepdim=True) / dim + EPS).sqrt()
            return c * w * q - x * q ** 3 * ((c * w * x).sum(1, keepdim=True) / dim), (c * x * q).sum(0), x * w * q
        total = f64(s["sum"])
        through, dw2, _ = back(f64(s["stream_out"]), w2 + o, f64(s["norm_grad"]))
        d = f64(s["stream_out_grad"]) + through
        out = {"stream": d, "pre_weight": dw2}
        c = scale * d if g is None else scale * d * g
        if w1 is None:
            out["send"], u = c, total
        else:
            out["send"], out["post_weight"], u = back(total, w1 + o, c)
        if g is not None:
            dg = scale * d * u
            if case["gate"] == "vector":
                out["gate"] = dg.sum(0)
            else:
                out["gate"] = torch.stack([part.sum(0) for part in dg.split(case["gate_rows"])]) if case["gate_rows"] > 1 else dg
        return out

    row = s["ids"].long() - case["first"]
    if case["op"] == "embed":
        out = torch.zeros((case["tokens"], case["dim"]), dtype=torch.float64, device="cuda")
        at = ((row >= 0) & (row < case["shard"])).nonzero()[:, 0]
        out[at] = f64(s["table"][row[at]]) * case["scale"]
        return out
    out = f64(s["table_grad"]) if case["accumulate"] else \
        torch.zeros((case["shard"], case["dim"]), dtype=torch.float64, device="cuda")
    at = ((row >= 0) & (row < case["shard"])).nonzero()[:, 0]
    return out.index_put_((row[at],), f64(s["out_grad"][at]) * case["scale"], accumulate=True)
