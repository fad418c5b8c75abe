"""Cases and plain forms of the row operators of language models.

Six operators on rows picked by index: the embedding lookup with a scale
("take") and its gradient by sorted tokens ("take_grad"), tokens sorted by
expert ("dispatch") and back with the router's weights ("combine"), and the
gradients of both ("dispatch_grad", "combine_grad").  An index outside its
range (a padded token, a dropped expert choice) picks nothing: its row is zero
and it has no gradient.

`own = False` computes them with elementary torch operations, `own = True`
through numba_mlir_b200.
"""

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_OPS = ("take", "take_grad", "dispatch", "combine", "dispatch_grad", "combine_grad")


# ------------------------------------------------------------------ cases ---
def _lookup(name, op, n, dim, rows, dtype, to, ids, dist="zipf", pad=0.0, scale=1.0, wide=0):
    """n tokens of a vocabulary of `rows`; `pad`: the share of them that is
    padding; `to`: the type of the result; `wide`: columns between the rows of
    the wider buffer that the table (the incoming gradient) is a slice of."""
    return {"name": name, "op": op, "n": n, "dim": dim, "rows": rows, "dtype": dtype, "to": to, "ids": ids,
            "dist": dist, "pad": pad, "scale": scale, "wide": wide}


def _routed(name, op, tokens, k, groups, dim, dtype, ids="i32", skew=0.5, drop=0.0, wide=0):
    """`tokens` tokens with k of `groups` experts each; `skew`: how uneven the
    experts are chosen; `drop`: the share of choices given up."""
    return {"name": name, "op": op, "tokens": tokens, "k": k, "groups": groups, "dim": dim, "dtype": dtype,
            "ids": ids, "skew": skew, "drop": drop, "wide": wide}


def listed():
    return [
        # one decoding step of sixteen sequences: latency
        _lookup("take-decode", "take", 16, 2048, 32768, "bf16", "bf16", "i64", scale=math.sqrt(2048.0)),
        # the prompts of a batch, or one training step's forward pass
        _lookup("take-prefill", "take", 16384, 4096, 131072, "bf16", "bf16", "i32", scale=64.0),
        # a small model of odd sizes trained in float32, a fifth of the batch padded
        _lookup("take_grad-odd", "take_grad", 777, 1000, 10007, "f32", "f32", "i64", pad=0.2, scale=0.5),
        # one training step: eight sequences of 4096 tokens
        _lookup("take_grad-train", "take_grad", 32768, 4096, 131072, "bf16", "bf16", "i32", scale=64.0),
        # a decoding step of four sequences through an expert layer: latency
        _routed("dispatch-decode", "dispatch", 4, 8, 64, 2048, "bf16"),
        # a prefill or training batch through an expert layer
        _routed("dispatch-train", "dispatch", 16384, 8, 128, 2048, "bf16"),
        # ragged everything: odd width, odd batch, some choices dropped at the experts' capacity
        _routed("combine-odd", "combine", 333, 3, 17, 1001, "f16", ids="i64", drop=0.1),
        # the way back of the training batch
        _routed("combine-train", "combine", 16384, 8, 128, 2048, "bf16"),
        # few large experts, float32, a few tokens per device, a narrow slice of a wider buffer
        _routed("dispatch_grad-small", "dispatch_grad", 300, 2, 8, 1024, "f32", wide=64),
        # backward pass of a training batch over wide rows, two experts each
        _routed("dispatch_grad-train", "dispatch_grad", 16384, 2, 16, 4096, "f16"),
        # a small batch with dropped choices
        _routed("combine_grad-small", "combine_grad", 1000, 6, 60, 1416, "bf16", ids="i64", drop=0.05),
        # backward pass of the training batch
        _routed("combine_grad-train", "combine_grad", 16384, 8, 128, 2048, "bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, hi):
    """A row's width: a multiple of 64, of 8, or any number."""
    w = _log(rng, 16, hi)
    step = rng.choice((64, 8, 1))
    return max(step, w // step * step)


def draw(rng):
    op = rng.choice(_OPS)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    ids = rng.choice(("i32", "i64"))
    wide = rng.choice((0, 0, 8, 3))
    gone = rng.choice((0.0, 0.0, rng.uniform(0.0, 0.5)))
    dim = _width(rng, 8192)
    if op in ("take", "take_grad"):
        to = dtype if rng.random() < 0.7 else ("f32" if dtype != "f32" else rng.choice(("bf16", "f16")))
        rows = min(_log(rng, 50, 200000), 131072 * 2048 // dim)
        n = min(_log(rng, 1, 65536), 16384 * 2048 // dim)
        return _lookup("", op, n, dim, max(1, rows), dtype, to, ids, rng.choice(("zipf", "uniform")), gone,
                       round(math.exp(rng.uniform(-3.0, 4.0)), 4), wide)
    groups = _log(rng, 2, 512)
    k = rng.choice([x for x in (1, 2, 3, 4, 6, 8, 10) if x <= groups])
    tokens = min(_log(rng, 1, 32768), max(1, 16384 * 2048 * 8 // 2 // (dim * k)))
    return _routed("", op, tokens, k, groups, dim, dtype, ids, rng.uniform(0.0, 1.5), gone, wide)


# ----------------------------------------------------------------- inputs ---
def _values(shape, dtype, gen, size, wide=0):
    """Normal values of standard deviation `size`, as a slice of a buffer that
    is `wide` columns wider."""
    full = (*shape[:-1], shape[-1] + wide)
    out = torch.empty(full, dtype=_DTYPES[dtype], device="cuda").normal_(0.0, size, generator=gen)
    return out[..., :shape[-1]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = torch.int64 if case["ids"] == "i64" else torch.int32
    dim = case["dim"]
    if case["op"] in ("take", "take_grad"):
        n, rows = case["n"], case["rows"]
        u = torch.rand(n, dtype=torch.float64, device="cuda", generator=gen)
        # zipf: the r-th most frequent token comes up about 1/r as often as the first
        at = (torch.exp(u * math.log(rows + 1.0)) - 1.0 if case["dist"] == "zipf" else u * rows)
        ids = at.to(torch.int64).clamp_(0, rows - 1)
        gone = torch.rand(n, device="cuda", generator=gen) < case["pad"]
        state = {"case": case, "ids": torch.where(gone, -1, ids).to(kind)}
        if case["op"] == "take":
            state["table"] = _values((rows, dim), case["dtype"], gen, 0.02, case["wide"])
        else:
            state["dout"] = _values((n, dim), case["dtype"], gen, 0.01, case["wide"])
        return state
    tokens, k, groups = case["tokens"], case["k"], case["groups"]
    liked = torch.randn(groups, device="cuda", generator=gen) * case["skew"]
    scores = torch.randn((tokens, groups), device="cuda", generator=gen) + liked
    best, ids = torch.topk(scores, k, dim=1)
    gone = torch.rand((tokens, k), device="cuda", generator=gen) < case["drop"]
    ids = torch.where(gone, -1, ids)
    if case["op"] == "dispatch":
        return {"case": case, "ids": ids.to(kind), "x": _values((tokens, dim), case["dtype"], gen, 1.0, case["wide"])}
    state = {"case": case, "weights": torch.softmax(best, dim=1)}
    # what the forward pass kept: where each choice went, and where each expert's rows begin
    key = torch.where(ids < 0, groups, ids).reshape(-1)
    ordered, order = torch.sort(key, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(tokens * k, device="cuda")
    state["order"] = order.to(torch.int32)
    state["place"] = place.to(torch.int32).reshape(tokens, k)
    state["offsets"] = torch.searchsorted(ordered, torch.arange(groups + 1, device="cuda")).to(torch.int32)
    if case["op"] != "dispatch_grad":
        state["ys"] = _values((tokens * k, dim), case["dtype"], gen, 1.0, case["wide"])
    if case["op"] == "combine_grad":
        state["dout"] = _values((tokens, dim), case["dtype"], gen, 0.01)
    if case["op"] == "dispatch_grad":
        state["dxs"] = _values((tokens * k, dim), case["dtype"], gen, 0.01, case["wide"])
    return state


# ------------------------------------------------------------- plain form ---
def _kept(ids, rows):
    return (ids >= 0) & (ids < rows)


def _plain_take(s):
    c, table = s["case"], s["table"]
    kept = _kept(s["ids"], c["rows"])
    picked = table[torch.where(kept, s["ids"], 0)].float() * c["scale"]
    return torch.where(kept[:, None], picked, 0.0).to(_DTYPES[c["to"]])


def _plain_take_grad(s):
    c = s["case"]
    at = torch.where(_kept(s["ids"], c["rows"]), s["ids"], c["rows"])
    total = torch.zeros((c["rows"] + 1, c["dim"]), device="cuda")
    total.index_add_(0, at, s["dout"].float())
    return (total[:c["rows"]] * c["scale"]).to(_DTYPES[c["to"]])


def _plain_dispatch(s):
    c, x = s["case"], s["x"]
    groups, n = c["groups"], c["tokens"] * c["k"]
    key = torch.where(_kept(s["ids"], groups), s["ids"], groups).reshape(-1)
    ordered, order = torch.sort(key, stable=True)
    at = torch.arange(n, device="cuda")
    place = torch.empty_like(order)
    place[order] = at
    offsets = torch.searchsorted(ordered, torch.arange(groups + 1, device="cuda", dtype=ordered.dtype))
    xs = torch.where((ordered < groups)[:, None], x[order // c["k"]], 0.0).to(x.dtype)
    return {"xs": xs, "order": order.to(torch.int32), "place": place.to(torch.int32).reshape(c["tokens"], c["k"]),
            "offsets": offsets.to(torch.int32)}


def _back(rows, place, offsets):
    """The rows of every token's choices, zero where the choice was dropped."""
    return torch.where((place < offsets[-1])[..., None], rows[place].float(), 0.0)


def _plain_combine(s):
    ys = s["ys"]
    return (_back(ys, s["place"], s["offsets"]) * s["weights"][..., None]).sum(1).to(ys.dtype)


def _plain_dispatch_grad(s):
    return _back(s["dxs"], s["place"], s["offsets"]).sum(1).to(s["dxs"].dtype)


def _plain_combine_grad(s):
    c, ys, place = s["case"], s["ys"], s["place"]
    d = s["dout"].float()[:, None, :]
    kept = place < s["offsets"][-1]
    dys = torch.empty((c["tokens"] * c["k"], c["dim"]), dtype=ys.dtype, device="cuda")
    dys[place] = torch.where(kept[..., None], s["weights"][..., None] * d, 0.0).to(ys.dtype)
    return {"dys": dys, "dweights": (_back(ys, place, s["offsets"]) * d).sum(-1)}


_PLAIN = {"take": _plain_take, "take_grad": _plain_take_grad, "dispatch": _plain_dispatch,
          "combine": _plain_combine, "dispatch_grad": _plain_dispatch_grad, "combine_grad": _plain_combine_grad}

# --------------------------------------------------- the framework's calls ---
_queue = None


def _on_stream(nm):
    """The queue of torch's current stream, made once as a program would."""
    global _queue
    if _queue is None:
        _queue = nm.runtime.Queue.from_stream(torch.cuda.current_stream().cuda_stream)
    return _queue


def _own_run(s):
    import numba_mlir_b200 as nm

    c, q = s["case"], _on_stream(nm)
    op, dim = c["op"], c["dim"]
    new = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    if op == "take":
        out = new((c["n"], dim), _DTYPES[c["to"]])
        nm.take_rows(s["table"], s["ids"], c["scale"], out=out, queue=q)
        return out
    if op == "take_grad":
        out = new((c["rows"], dim), _DTYPES[c["to"]])
        nm.take_rows_grad(s["dout"], s["ids"], scale=c["scale"], out=out, queue=q)
        return out
    tokens, k = c["tokens"], c["k"]
    if op == "dispatch":
        xs = new((tokens * k, dim), s["x"].dtype)
        order, place = new((tokens * k,), torch.int32), new((tokens, k), torch.int32)
        offsets = new((c["groups"] + 1,), torch.int32)
        nm.dispatch_rows(s["x"], s["ids"], c["groups"], out=xs, plan=nm.RowGroups(order, place, offsets), queue=q)
        return {"xs": xs, "order": order, "place": place, "offsets": offsets}
    plan = nm.RowGroups(s["order"], s["place"], s["offsets"])
    if op == "combine":
        out = new((tokens, dim), s["ys"].dtype)
        nm.combine_rows(s["ys"], plan, s["weights"], out=out, queue=q)
        return out
    if op == "dispatch_grad":
        out = new((tokens, dim), s["dxs"].dtype)
        nm.dispatch_rows_grad(s["dxs"], plan, out=out, queue=q)
        return out
    dys, dweights = new((tokens * k, dim), s["ys"].dtype), new((tokens, k), torch.float32)
    nm.combine_rows_grad(s["dout"], s["ys"], plan, s["weights"], out=dys, dweights=dweights, queue=q)
    return {"dys": dys, "dweights": dweights}


def run(state):
    return _own_run(state) if own else _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------- work ---
def work(case):
    """Each input row read once, each output row written once, and the indices."""
    size, dim = _SIZE[case["dtype"]], case["dim"]
    index = 8 if case["ids"] == "i64" else 4
    if case["op"] in ("take", "take_grad"):
        n, to = case["n"], _SIZE[case["to"]]
        live = n * (1.0 - case["pad"])
        if case["op"] == "take":
            # a token that comes up again is read from memory once
            rows = case["rows"]
            if case["dist"] == "uniform":
                seen = rows * (1.0 - math.exp(-live / rows))
            else:
                # the r-th token has probability log((r + 1) / r) / log(rows + 1)
                seen, low = 0.0, 1
                while low <= rows:
                    high = min(rows + 1, max(low + 1, low * 5 // 4))
                    p = math.log(high / low) / math.log(rows + 1.0) / (high - low)
                    seen += (high - low) * (1.0 - math.exp(-live * p))
                    low = high
            return {"bytes": seen * dim * size + n * (dim * to + index), "flops": live * dim}
        return {"bytes": n * index + live * dim * size + case["rows"] * dim * to, "flops": live * dim}
    tokens, k = case["tokens"], case["k"]
    n = tokens * k
    live = n * (1.0 - case["drop"])
    rows, token_rows = live * dim * size, tokens * dim * size
    if case["op"] == "dispatch":
        return {"bytes": token_rows + n * dim * size + n * (index + 8) + case["groups"] * 4, "flops": 0}
    if case["op"] == "combine":
        return {"bytes": rows + token_rows + n * 8, "flops": 2 * live * dim}
    if case["op"] == "dispatch_grad":
        return {"bytes": rows + token_rows + n * 4, "flops": live * dim}
    return {"bytes": rows + token_rows + n * dim * size + n * 12, "flops": 3 * live * dim}


# ------------------------------------------------------------------ exact ---
def exact(case, seed):
    """The definitions in float64, one row or one choice at a time."""
    s = prepare(case, seed)
    op, dim = case["op"], case["dim"]
    if op in ("take", "take_grad"):
        ids = s["ids"].to(torch.int64)
        live = torch.nonzero((ids >= 0) & (ids < case["rows"]))[:, 0]
        if op == "take":
            out = torch.zeros((case["n"], dim), dtype=torch.float64, device="cuda")
            out[live] = torch.index_select(s["table"], 0, ids[live]).double() * case["scale"]
            return out
        out = torch.zeros((case["rows"], dim), dtype=torch.float64, device="cuda")
        out.index_put_((ids[live],), s["dout"][live].double() * case["scale"], accumulate=True)
        return out
    tokens, k, groups = case["tokens"], case["k"], case["groups"]
    if op == "dispatch":
        choice = s["ids"].reshape(-1).cpu().to(torch.int64)
        found = [torch.nonzero(choice == g)[:, 0] for g in range(groups)]
        lost = torch.nonzero((choice < 0) | (choice >= groups))[:, 0]
        order = torch.cat(found + [lost])
        offsets = torch.tensor([0] + [len(f) for f in found]).cumsum(0)
        place = torch.argsort(order)
        xs = torch.zeros((tokens * k, dim), dtype=torch.float64, device="cuda")
        live = int(offsets[-1])
        xs[:live] = s["x"].double()[torch.div(order[:live], k, rounding_mode="floor").cuda()]
        return {"xs": xs, "order": order.to(torch.int32), "place": place.to(torch.int32).reshape(tokens, k),
                "offsets": offsets.to(torch.int32)}
    place, live = s["place"].to(torch.int64), int(s["offsets"][-1])
    weights = s["weights"].double() if op != "dispatch_grad" else torch.ones((tokens, k), dtype=torch.float64, device="cuda")
    if op in ("combine", "dispatch_grad"):
        rows = s["ys"] if op == "combine" else s["dxs"]
        out = torch.zeros((tokens, dim), dtype=torch.float64, device="cuda")
        for j in range(k):
            here = torch.nonzero(place[:, j] < live)[:, 0]
            out[here] += weights[here, j, None] * rows[place[here, j]].double()
        return out
    dys = torch.zeros((tokens * k, dim), dtype=torch.float64, device="cuda")
    dweights = torch.zeros((tokens, k), dtype=torch.float64, device="cuda")
    d = s["dout"].double()
    for j in range(k):
        here = torch.nonzero(place[:, j] < live)[:, 0]
        dys[place[here, j]] = weights[here, j, None] * d[here]
        dweights[here, j] = torch.linalg.vecdot(s["ys"][place[here, j]].double(), d[here])
    return {"dys": dys, "dweights": dweights}
