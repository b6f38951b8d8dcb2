"""What the operators from the router to the loss are timed on: those that stand before, between and behind a
model's products.

A case is one pass through one operator, as a program calls it through ``Loader``:

``route``               the experts of every token and their weights, from the router's logits
``dispatch``            the rows of the tokens sorted by expert, and the row offsets that ``grouped`` reads
``combine``             the experts' rows summed by token with the router's weights
``cross_entropy``       the loss of a projection onto a vocabulary, without keeping its logits
``distillation``        the same against the listed logits of a teacher

With ``step`` the pass is one of training: the operator and its gradients.  Sizes are those of the library's own
configurations, tests and benchmark, or generic; ``draw`` spreads over the same ranges.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
MOST_FLOPS = 7e12  # no drawn case costs more than the largest listed one
MOST_BYTES = 1.5e9


def _route(m, experts, k, logits, score, bias=False, groups=1, kept=1, best=2, renormalize=True, scale=1.0, padding=0.0,
           step=False):
    """kept: groups that a token may choose from; best: how many of a group's experts make its score; padding: the share
    of the tokens that go nowhere."""
    return {"kind": "route", "m": m, "experts": experts, "k": k, "logits": logits, "score": score, "bias": bias,
            "groups": groups, "kept": kept, "best": best, "renormalize": renormalize, "scale": scale, "padding": padding,
            "step": step}


def _rows(kind, m, n, k, experts, rows, weights=True, residual=False, padding=0.0, routing=0, step=False):
    """routing: a seed; which experts the tokens choose follows from it, the sizes and the share of padding."""
    return {"kind": kind, "m": m, "n": n, "k": k, "experts": experts, "rows": rows, "weights": weights,
            "residual": residual, "padding": padding, "routing": routing, "step": step}


def _loss(kind, m, n, k, ab, layout="c", entries=0, temperature=1.0, ignored=0.1, step=False):
    """layout: of B (K x N); c = column-major, weights stored N x K, r = row-major.  ignored: the share of the rows
    that have no target."""
    return {"kind": kind, "m": m, "n": n, "k": k, "ab": ab, "layout": layout, "entries": entries,
            "temperature": temperature, "ignored": ignored, "step": step}


def listed():
    return [
        # one token of a decode through a router: a call's latency
        dict(_route(1, 64, 2, "f32", "softmax"), name="route_token_1x64_2_f32"),
        # prefill of an odd number of tokens over many small experts in groups, balanced by a bias
        dict(_route(8191, 256, 8, "f32", "sigmoid", bias=True, groups=8, kept=4, scale=2.5),
             name="route_prefill_8191x256_8_grouped_f32"),
        # training: the choice and the gradient of the logits, padded batch
        dict(_route(16384, 128, 8, "bf16", "softmax", padding=0.05, step=True), name="route_step_16384x128_8_bf16"),
        # decode: a batch of sequences to their experts
        dict(_rows("dispatch", 32, 4096, 8, 64, "bf16", routing=1), name="dispatch_decode_32x4096_8_of_64_bf16"),
        # training: an odd number of tokens to many experts
        dict(_rows("dispatch", 8191, 2048, 6, 128, "bf16", routing=2), name="dispatch_train_8191x2048_6_of_128_bf16"),
        # one token back from its experts, onto the residual stream
        dict(_rows("combine", 1, 5120, 8, 64, "f16", residual=True, routing=3), name="combine_token_1x5120_8_f16"),
        # training: back from the experts, and the gradients of their rows and weights
        dict(_rows("combine", 8192, 4096, 4, 32, "bf16", padding=0.05, routing=4, step=True),
             name="combine_step_8192x4096_4_bf16"),
        # the likelihood of a short answer: the vocabulary's weights from memory
        dict(_loss("cross_entropy", 17, 50001, 2048, "f16"), name="cross_entropy_17x50001x2048_f16"),
        # training: the loss of a batch and the gradients of the projection
        dict(_loss("cross_entropy", 4096, 65536, 4096, "bf16", step=True), name="cross_entropy_step_4096x65536x4096_bf16"),
        # odd in every extent, weights stored K x N
        dict(_loss("cross_entropy", 1999, 32003, 999, "f16", layout="r", step=True),
             name="cross_entropy_step_1999x32003x999_f16"),
        # how far a student is from its teacher
        dict(_loss("distillation", 2048, 65536, 2048, "bf16", entries=32, temperature=2.0),
             name="distillation_2048x65536x2048_32_bf16"),
        # training a student on its teacher's best logits
        dict(_loss("distillation", 1001, 32000, 1024, "f16", entries=64, temperature=1.0, step=True),
             name="distillation_step_1001x32000x1024_64_f16"),
    ]


def _spread(rng, low, high, grain=1):
    """A size between low and high, spread over its logarithm, a multiple of grain."""
    return max(grain, int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / grain)) * grain)


def draw(rng):
    kind = rng.choice(("route", "route", "dispatch", "combine", "combine", "cross_entropy", "cross_entropy", "distillation"))
    if kind == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        each = max(4, _spread(rng, 8, 512) // groups)
        experts, kept = groups * each, rng.randint(1, groups)
        score = rng.choice(("softmax", "sigmoid"))
        return _route(_spread(rng, 1, 32768), experts, rng.randint(1, min(16, kept * each)), rng.choice(("f32", "bf16", "f16")),
                      score, bias=rng.random() < 0.5, groups=groups, kept=kept, best=rng.randint(1, 2),
                      renormalize=rng.random() < 0.7, scale=rng.choice((1.0, 2.5)), padding=rng.choice((0.0, 0.1)),
                      step=rng.random() < 0.5)
    if kind in ("dispatch", "combine"):
        experts = _spread(rng, 2, 256)
        k = rng.randint(1, min(8, experts))
        rows = rng.choice(("bf16", "bf16", "f16", "f32"))
        n = _spread(rng, 256, 8192, rng.choice((64, 64, 8, 1)))
        m = _spread(rng, 1, 16384)
        while m * n * (2 * k + 1) * (4 if rows == "f32" else 2) > MOST_BYTES:
            m = max(1, m // 2)
        return _rows(kind, m, n, k, experts, rows, weights=rng.random() < 0.8, residual=rng.random() < 0.3,
                     padding=rng.choice((0.0, 0.1)), routing=rng.randrange(1 << 20),
                     step=kind == "combine" and rng.random() < 0.5)
    grain = rng.choice((64, 64, 8, 1))
    n, k = _spread(rng, 1024, 131072, grain), _spread(rng, 256, 8192, grain)
    step = rng.random() < 0.6
    m = _spread(rng, 1, 8192) if rng.random() < 0.7 else _spread(rng, 1, 127)
    while (8.0 if step else 2.0) * m * n * k > MOST_FLOPS:
        m = max(1, m // 2)
    while n * k > 1 << 29:
        n = max(grain, n // 2 // grain * grain)
    entries = 0 if kind == "cross_entropy" else _spread(rng, 4, 128)
    return _loss(kind, m, n, k, rng.choice(("bf16", "f16")), rng.choice("ccr"), entries,
                 1.0 if not entries else rng.choice((1.0, 2.0, 4.0)), rng.choice((0.0, 0.1, 0.5)), step)


def _normal(generator, shape, dtype, scale=1.0):
    x = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, scale, generator=generator)
    return x.to(dtype)


def _uniform(generator, shape):
    return torch.rand(shape, dtype=torch.float32, device="cuda", generator=generator)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = dict(case)
    if own:
        import rocm_wmma_gemm_amd as R

        state["loader"] = R.Loader()
        state["codes"] = {"r": R.row_major, "c": R.col_major}
        state["scores"] = {"softmax": R.score.softmax, "sigmoid": R.score.sigmoid}
    new = lambda shape, dtype: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    m, k = case["m"], case["k"]
    if case["kind"] == "route":
        e, logits = case["experts"], DTYPES[case["logits"]]
        state["x"] = _normal(g, (m, e), logits, 1.5)
        # (what keeps the experts' loads equal is of the size of the scores' differences)
        state["balance"] = _normal(g, (e,), torch.float32, 0.05 if case["score"] == "sigmoid" else 0.01) if case["bias"] else None
        state["real"] = _uniform(g, (m,)) >= case["padding"] if case["padding"] else None
        state["dweights"] = _normal(g, (m, k), torch.float32) if case["step"] else None
        state["chosen"], state["weights"] = new((m, k), torch.int32), new((m, k), torch.float32)
        state["dx"] = new((m, e), logits) if case["step"] else None
        return state
    if case["kind"] in ("dispatch", "combine"):
        n, e, rows = case["n"], case["experts"], DTYPES[case["rows"]]
        popular = torch.Generator(device="cuda")
        popular.manual_seed(case["routing"])
        # k different experts for every token, some more popular than others
        liked = _normal(popular, (e,), torch.float32) - torch.log(-torch.log(_uniform(g, (m, e)).clamp(1e-7, 1 - 1e-7)))
        state["chosen"] = liked.argsort(1, descending=True)[:, :k].to(torch.int32).contiguous()
        if case["padding"]:
            state["chosen"][_uniform(g, (m,)) < case["padding"]] = -1
        state["places"], state["offsets"] = new((m, k), torch.int32), new((e + 1,), torch.int32)
        if case["kind"] == "dispatch":
            state["x"], state["rows_out"] = _normal(g, (m, n), rows), new((m * k, n), rows)
            return state
        state["places"] = _sorted_places(state["chosen"], e)[0]
        state["y"] = _normal(g, (m * k, n), rows)
        state["weights_in"] = _uniform(g, (m, k)) / k if case["weights"] else None
        state["residual_in"] = _normal(g, (m, n), rows) if case["residual"] else None
        state["out"] = new((m, n), rows)
        if case["step"]:
            state["dout"], state["dy"] = _normal(g, (m, n), rows), new((m * k, n), rows)
            state["dweights"] = new((m, k), torch.float32) if case["weights"] else None
        return state
    n, ab, entries = case["n"], DTYPES[case["ab"]], case["entries"]
    b = _normal(g, (n, k), ab, 2.0 / math.sqrt(k))
    targets = torch.randint(n, (m,), device="cuda", generator=g)
    ignored = _uniform(g, (m,)) < case["ignored"]
    # states that lean towards their targets, some more than others
    state["a"] = (_normal(g, (m, k), torch.float32) + 3.0 * _uniform(g, (m, 1)) * b[targets].float()).to(ab)
    state["b"] = b if case["layout"] == "c" else b.t().contiguous()
    if entries:
        # a teacher's best: different entries, the target's first; short lists end in -1
        first = torch.randint(n, (m, 1), device="cuda", generator=g)
        hop = torch.randint(1, max(2, n // entries), (m, 1), device="cuda", generator=g)
        state["listed"] = (first + hop * torch.arange(entries, device="cuda")) % n
        state["listed"][:, entries // 2:][_uniform(g, (m,)) < 0.1] = -1
        state["listed"][ignored] = -1
        state["listed"] = state["listed"].to(torch.int32)
        state["teacher"] = _normal(g, (m, entries), torch.float32, 2.0).sort(1, descending=True)[0] + 4.0
        state["picked"] = new((m, entries), torch.float32)
    else:
        state["targets"] = torch.where(ignored, torch.full_like(targets, -100), targets)
    state["loss"], state["lse"] = new((m,), torch.float32), new((m,), torch.float32)
    if case["step"]:
        # the mean over the rows that count; training in f16 scales its loss
        count = max(1.0, float((~ignored).sum()))
        state["dloss"] = (~ignored).float() * ((4096.0 if case["ab"] == "f16" else 1.0) / count)
        state["da"], state["db"] = new((m, k), ab), new(state["b"].shape, ab)
    return state


def _run_own(s):
    loader, m, k = s["loader"], s["m"], s["k"]
    if s["kind"] == "route":
        score = s["scores"][s["score"]]
        loader.route(s["chosen"], s["weights"], s["x"], m, s["experts"], k, score=score, bias=s["balance"], mask=s["real"],
                     groups=s["groups"], kept_groups=s["kept"], group_best=s["best"], renormalize=s["renormalize"],
                     scale=s["scale"])
        if s["step"]:
            loader.route_backward(s["dx"], s["dweights"], s["chosen"], s["x"], m, s["experts"], k, score=score,
                                  renormalize=s["renormalize"], scale=s["scale"])
        return [s["chosen"], s["weights"], s["dx"]]
    n = s["n"]
    if s["kind"] == "dispatch":
        loader.dispatch(s["rows_out"], s["offsets"], s["places"], s["x"], s["chosen"], m, n, k)
        return [s["rows_out"], s["offsets"], s["places"]]
    if s["kind"] == "combine":
        loader.combine(s["out"], s["y"], s["places"], m, n, k, weights=s["weights_in"], residual=s["residual_in"])
        if not s["step"]:
            return [s["out"]]
        loader.combine_backward(s["dy"], s["dweights"], s["dout"], s["y"], s["places"], m, n, k, weights=s["weights_in"])
        return [s["out"], s["dy"], s["dweights"]]
    layout = s["codes"][s["layout"]]
    if s["entries"]:
        loader.linear_distillation(s["loss"], s["lse"], s["picked"], s["a"], s["b"], s["listed"], s["teacher"], m, n, k,
                                   layout, temperature=s["temperature"])
        if s["step"]:
            loader.linear_distillation_backward(s["da"], s["db"], s["dloss"], s["lse"], s["picked"], s["a"], s["b"],
                                                s["listed"], s["teacher"], m, n, k, layout, temperature=s["temperature"])
    else:
        loader.linear_cross_entropy(s["loss"], s["lse"], s["a"], s["b"], s["targets"], m, n, k, layout)
        if s["step"]:
            loader.linear_cross_entropy_backward(s["da"], s["db"], s["dloss"], s["lse"], s["a"], s["b"], s["targets"],
                                                 m, n, k, layout)
    return [s["loss"], s["lse"]] + ([s["da"], s["db"]] if s["step"] else [])


def _sorted_places(chosen, experts):
    """Where every choice's row lies when the choices are sorted by expert, in their order within one; the experts' ends."""
    flat = chosen.flatten().long()
    flat = torch.where(flat < 0, experts, flat)
    order = torch.argsort(flat, stable=True)
    places = torch.empty_like(flat)
    places[order] = torch.arange(flat.numel(), device="cuda")
    places = torch.where(flat < experts, places, -1).to(torch.int32).view(chosen.shape)
    offsets = torch.searchsorted(flat[order], torch.arange(experts + 1, device="cuda")).to(torch.int32)
    return places, offsets, order


def run(state):
    if own:
        return _run_own(state)
    return {"route": _plain_route, "dispatch": _plain_dispatch, "combine": _plain_combine, "cross_entropy": _plain_loss,
            "distillation": _plain_loss}[state["kind"]](state)


def _scores(x, score):
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    e = torch.exp(x - x.max(1, keepdim=True)[0])
    return e / e.sum(1, keepdim=True)


def _plain_route(s):
    m, e, k = s["m"], s["experts"], s["k"]
    x = s["x"].double()  # (two scores next to each other are told apart)
    p = _scores(x, s["score"])
    value = p if s["balance"] is None else p + s["balance"].double()
    key = x if s["balance"] is None else value
    if s["groups"] > 1:
        size = e // s["groups"]
        of_group = value.view(m, s["groups"], size).sort(2, descending=True)[0][:, :, :s["best"]].sum(2)
        kept = of_group.sort(dim=1, descending=True, stable=True)[1][:, :s["kept"]]
        allowed = torch.zeros((m, s["groups"]), dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        key = torch.where(allowed.repeat_interleave(size, 1), key, -math.inf)
    chosen = key.sort(dim=1, descending=True, stable=True)[1][:, :k]
    w = p.gather(1, chosen)
    total = w.sum(1, keepdim=True) if s["renormalize"] else torch.ones_like(w[:, :1])
    w = w / total * s["scale"]
    real = torch.ones((m, 1), dtype=torch.bool, device="cuda") if s["real"] is None else s["real"][:, None]
    dx = None
    if s["step"]:
        dw = s["dweights"].double()
        ds = s["scale"] * dw / total
        if s["renormalize"]:
            ds = ds - (dw * w).sum(1, keepdim=True) / total
        ds = torch.zeros_like(p).scatter_(1, chosen, ds)
        dx = ds * p * (1.0 - p) if s["score"] == "sigmoid" else p * (ds - (ds * p).sum(1, keepdim=True))
        dx = torch.where(real, dx, 0.0).to(s["x"].dtype)
    return [torch.where(real, chosen, -1).to(torch.int32), torch.where(real, w, 0.0).float(), dx]


def _plain_dispatch(s):
    places, offsets, order = _sorted_places(s["chosen"], s["experts"])
    rows = s["x"][order // s["k"]]
    used = torch.arange(rows.shape[0], device="cuda") < offsets[-1]
    return [torch.where(used[:, None], rows, 0), offsets, places]


def _plain_combine(s):
    there = (s["places"] >= 0)[:, :, None]
    y = torch.where(there, s["y"][s["places"].clamp_min(0).long()].float(), 0.0)
    w = torch.ones_like(y[:, :, :1]) if s["weights_in"] is None else s["weights_in"][:, :, None]
    out = (w * y).sum(1)
    if s["residual_in"] is not None:
        out = out + s["residual_in"].float()
    out = out.to(s["y"].dtype)
    if not s["step"]:
        return [out]
    dout = s["dout"].float()[:, None, :]
    dy = torch.zeros((s["m"] * s["k"] + 1, s["n"]), dtype=torch.float32, device="cuda")
    dy[torch.where(s["places"] >= 0, s["places"], s["m"] * s["k"]).long()] = w * dout
    dweights = None if s["weights_in"] is None else (dout * y).sum(2)
    return [out, dy[:-1].to(s["y"].dtype), dweights]


def _plain_loss(s):
    a, b, t = s["a"].float(), s["b"].float(), s["temperature"]
    b = b.t() if s["layout"] == "c" else b
    z = a @ b / t
    top = z.max(1, keepdim=True)[0]
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    if s["entries"]:
        there = s["listed"] >= 0
        at = s["listed"].clamp_min(0).long()
        given = torch.where(there, s["teacher"] / t, -math.inf)
        most = given.max(1, keepdim=True)[0].clamp_min(-1e30)
        q = torch.exp(given - most)
        total = q.sum(1, keepdim=True)
        q = torch.where(total > 0, q / total, 0.0)
        log_q = torch.where(there, given - most - torch.log(total), 0.0)
        loss = t * t * (q * torch.where(there, log_q - (z.gather(1, at) - lse), 0.0)).sum(1)
        real = total > 0
    else:
        real = (s["targets"] >= 0)[:, None]
        at = s["targets"].clamp_min(0)[:, None]
        q = real.float()
        loss = torch.where(real, lse - z.gather(1, at), 0.0)[:, 0]
    if not s["step"]:
        return [loss, lse[:, 0]]
    p = torch.where(real, torch.exp(z - lse), 0.0)
    dz = t * s["dloss"][:, None] * p.scatter_add(1, at, -q)
    da, db = dz @ b.t(), a.t() @ dz
    if s["layout"] == "c":
        db = db.t().contiguous()
    return [loss, lse[:, 0], da.to(s["a"].dtype), db.to(s["a"].dtype)]


def work(case):
    m, k = case["m"], case["k"]
    if case["kind"] == "route":
        size, e = (4 if case["logits"] == "f32" else 2), case["experts"]
        # read, chosen and weights written; back: read again with the weights' gradients, written
        once = m * e * size + 8 * m * k + (4 * e if case["bias"] else 0)
        back = m * e * 2 * size + 8 * m * k if case["step"] else 0
        # an exponential is counted as ten operations, a comparison with the best so far as one for each choice
        return {"bytes": once + back, "flops": float(m * e * (10 + k) * (2 if case["step"] else 1))}
    if case["kind"] in ("dispatch", "combine"):
        n, size = case["n"], 4 if case["rows"] == "f32" else 2
        real = m * (1.0 - case["padding"])
        if case["kind"] == "dispatch":
            return {"bytes": size * n * real * (1 + k) + 8 * m * k + 4 * case["experts"], "flops": 4.0 * m * k}
        listed = 4 * m * k * (2 if case["weights"] else 1)
        once = size * n * (real * k + m * (2 if case["residual"] else 1)) + listed
        back = size * n * (real * k * (2 if case["weights"] else 1) + m) + listed + 4 * m * k if case["step"] else 0
        return {"bytes": once + back, "flops": float(real * n * k * (2 + (3 if case["step"] else 0)))}
    n, lists = case["n"], 8 * m * max(1, case["entries"])
    operands = 2 * (m * k + n * k)
    if not case["step"]:
        return {"bytes": operands + lists + 8 * m, "flops": 2.0 * m * n * k}
    # the logits once for the loss, once more for the gradient, and its two products
    return {"bytes": 2 * operands + 2 * lists + 12 * m, "flops": 8.0 * m * n * k}


def exact(case, seed):
    """What run() returns for these inputs by the definitions in 64 bits."""
    s = prepare(case, seed)
    return {"route": _exact_route, "dispatch": _exact_dispatch, "combine": _exact_combine, "cross_entropy": _exact_loss,
            "distillation": _exact_loss}[case["kind"]](s)


def _exact_route(s):
    m, e, k, groups = s["m"], s["experts"], s["k"], s["groups"]
    x = s["x"].double()
    p = torch.sigmoid(x) if s["score"] == "sigmoid" else torch.softmax(x, 1)
    value = p if s["balance"] is None else p + s["balance"].double()
    rank = (x if s["balance"] is None else value).clone()
    if groups > 1:
        best = torch.stack([v.topk(min(s["best"], e // groups), 1)[0].sum(1) for v in value.split(e // groups, 1)], 1)
        # a group stays where fewer than `kept` are better, or as good and before it
        ahead = torch.stack([(best > best[:, [g]]).sum(1) + (best[:, :g] == best[:, [g]]).sum(1) for g in range(groups)], 1)
        for g in range(groups):
            rank[:, g * (e // groups):(g + 1) * (e // groups)][ahead[:, g] >= s["kept"]] = -math.inf
    chosen = torch.empty((m, k), dtype=torch.int64, device="cuda")
    for j in range(k):
        top = rank.max(1, keepdim=True)[0]
        first = torch.where(rank == top, torch.arange(e, device="cuda"), e).min(1)[0]
        chosen[:, j] = first
        rank[torch.arange(m, device="cuda"), first] = -math.inf
    picked = p.gather(1, chosen)
    w = s["scale"] * (picked / picked.sum(1, keepdim=True) if s["renormalize"] else picked)
    dx = None
    if s["step"]:
        # by the chain of derivatives: weights by scores, scores by logits, written out
        total = picked.sum(1, keepdim=True)
        if s["renormalize"]:
            by_score = s["scale"] * (s["dweights"].double() * total - (s["dweights"].double() * picked).sum(1, keepdim=True)) / total ** 2
        else:
            by_score = s["scale"] * s["dweights"].double()
        full = torch.zeros_like(p)
        full.scatter_add_(1, chosen, by_score)
        dx = full * torch.exp(-x.abs()) / (1 + torch.exp(-x.abs())) ** 2 if s["score"] == "sigmoid" else \
            full * p - p * (by_score * picked).sum(1, keepdim=True)
    if s["real"] is not None:
        chosen[~s["real"]] = -1
        w[~s["real"]] = 0
        if dx is not None:
            dx[~s["real"]] = 0
    return [chosen.to(torch.int32), w, dx]


def _exact_dispatch(s):
    m, k, e = s["m"], s["k"], s["experts"]
    flat = s["chosen"].flatten().cpu()
    rows, offsets, places, at = torch.zeros((m * k, s["n"]), dtype=torch.float64, device="cuda"), [0], torch.full((m * k,), -1), 0
    for i in range(e):
        here = (flat == i).nonzero()[:, 0]
        places[here] = torch.arange(at, at + here.numel())
        rows[at:at + here.numel()] = s["x"][(here // k).cuda()].double()
        at += here.numel()
        offsets.append(at)
    return [rows, torch.tensor(offsets, dtype=torch.int32, device="cuda"), places.to(torch.int32).view(m, k).cuda()]


def _exact_combine(s):
    m, n, k = s["m"], s["n"], s["k"]
    out = torch.zeros((m, n), dtype=torch.float64, device="cuda") if s["residual_in"] is None else s["residual_in"].double()
    dy = torch.zeros((m * k, n), dtype=torch.float64, device="cuda")
    dweights = torch.zeros((m, k), dtype=torch.float64, device="cuda")
    for j in range(k):
        tokens = (s["places"][:, j] >= 0).nonzero()[:, 0]
        at = s["places"][tokens, j].long()
        w = 1.0 if s["weights_in"] is None else s["weights_in"][tokens, j].double()[:, None]
        out[tokens] += w * s["y"][at].double()
        if s["step"]:
            dy[at] = w * s["dout"][tokens].double()
            dweights[tokens, j] = torch.linalg.vecdot(s["dout"][tokens].double(), s["y"][at].double())
    if not s["step"]:
        return [out]
    return [out, dy, None if s["weights_in"] is None else dweights]


def _exact_loss(s):
    """Row by row of the softmax, some hundred rows at a time."""
    m, n, t = s["m"], s["n"], s["temperature"]
    b = s["b"].double()
    b = b if s["layout"] == "c" else b.t()  # n x k
    loss, lse = (torch.zeros((m,), dtype=torch.float64, device="cuda") for _ in range(2))
    da, db = torch.zeros(s["a"].shape, dtype=torch.float64, device="cuda"), torch.zeros((n, s["k"]), dtype=torch.float64, device="cuda")
    for first in range(0, m, 512):
        rows = slice(first, min(m, first + 512))
        a = s["a"][rows].double()
        lse[rows] = torch.logsumexp(a @ b.t() / t, 1)
        log_p = a @ b.t() / t - lse[rows, None]
        q = torch.zeros_like(log_p)
        if s["entries"]:
            at = s["listed"][rows].long()
            of = torch.softmax(torch.where(at >= 0, s["teacher"][rows].double() / t, -math.inf), 1).nan_to_num(0.0)
            q.scatter_add_(1, at.clamp_min(0), of)
            log_of = torch.where(of > 0, of.log(), 0.0)
            loss[rows] = t * t * (of * (log_of - log_p.gather(1, at.clamp_min(0)))).sum(1)
        else:
            at = s["targets"][rows]
            q[at >= 0, at[at >= 0]] = 1.0
            loss[rows] = -(q * log_p).sum(1)
        if s["step"]:
            dz = (log_p.exp() * (q.sum(1, keepdim=True) > 0) - q) * t * s["dloss"][rows].double()[:, None]
            da[rows] = dz @ b
            db += dz.t() @ a
    if not s["step"]:
        return [loss, lse]
    return [loss, lse, da, db if s["layout"] == "c" else db.t().contiguous()]
