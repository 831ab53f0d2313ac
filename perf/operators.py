"""The minibatch operators on factor tables, as a training or serving loop calls them: table lookup with scaling and its
gradient, the softmax loss over a catalogue of items with its gradient, and the clipping of gradients by their global
norm.  Widths and table heights are those of the rating sets the benchmark knows (workloads.py)."""
import torch

own = False

# rows of the user or item tables of the benchmark's rating sets, and the widths used with them
_HEIGHTS = (943, 1682, 3706, 6040, 17770, 59047, 162541, 480189, 624961)
_WIDTHS = (32, 40, 64, 128, 256)
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # the users of one small request, looked up for scoring: latency
        {"name": "lookup_request_f32", "op": "lookup", "n": 32, "rows": 480189, "d": 128, "type": "f32"},
        # the items of many histories at once, bf16 rows of 200 bytes
        {"name": "lookup_histories_bf16", "op": "lookup", "n": 1000003, "rows": 59047, "d": 100, "type": "bf16"},
        # gradient of a small batch of a small catalogue
        {"name": "lookup_grad_small_f32", "op": "lookup_grad", "n": 1000, "rows": 1682, "d": 32, "type": "f32"},
        # an ordinary training batch of histories: popular items occur thousands of times
        {"name": "lookup_grad_batch_bf16", "op": "lookup_grad", "n": 131072, "rows": 59047, "d": 128, "type": "bf16"},
        # a large accumulated batch against the largest user table of the fp32 benchmark
        {"name": "lookup_grad_large_f32", "op": "lookup_grad", "n": 2000003, "rows": 480189, "d": 128, "type": "f32"},
        # the loss of one request while serving
        {"name": "loss_one_f32", "op": "loss", "n": 1, "rows": 17770, "d": 128, "type": "f32", "bias": True},
        # held-out evaluation, odd batch, rows that are no multiple of 16 bytes
        {"name": "loss_heldout_bf16", "op": "loss", "n": 5003, "rows": 59047, "d": 100, "type": "bf16", "bias": False},
        # a training step at the model's default width on a small catalogue
        {"name": "train_default_f32", "op": "train", "n": 1000, "rows": 3706, "d": 40, "type": "f32", "bias": True, "weighted": False},
        # an ordinary training step in the tables' own type
        {"name": "train_batch_f32", "op": "train", "n": 8192, "rows": 17770, "d": 128, "type": "f32", "bias": True, "weighted": True},
        # the largest catalogue and width of the benchmark's rating sets, in bf16
        {"name": "train_large_bf16", "op": "train", "n": 4096, "rows": 624961, "d": 256, "type": "bf16", "bias": True, "weighted": False},
        # clipping of a small model's gradients: latency
        {"name": "clip_small_f32", "op": "clip", "rows": 6040, "cols": 3706, "d": 64, "pieces": 1, "type": "f32", "clipped": True},
        # clipping of a large model's gradients: bandwidth
        {"name": "clip_large_f32", "op": "clip", "rows": 480189, "cols": 17770, "d": 128, "pieces": 1, "type": "f32", "clipped": True},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "loss", "train", "train", "clip"])
    kind = rng.choice(["f32", "bf16"])
    d = rng.choice(_WIDTHS) if rng.random() < 0.5 else rng.randint(16, 256)
    rows = rng.choice(_HEIGHTS) if rng.random() < 0.5 else _spread(rng, 100, 624961)
    if op in ("lookup", "lookup_grad"):
        n = _spread(rng, 1, 2000003)
        return {"op": op, "n": max(1, min(n, 2000003 * 128 // d)), "rows": max(100, min(rows, 480189 * 128 // d)), "d": d, "type": kind}
    if op == "clip":
        return {"op": op, "rows": min(rows, 480189 * 128 // d), "cols": _spread(rng, 100, 17770), "d": d,
                "pieces": _spread(rng, 1, 300), "type": kind, "clipped": rng.random() < 0.5}
    n = _spread(rng, 1, 8192)
    most = 4096 * 624961 * 256 // (4 if kind == "f32" else 1)     # fp32 products take longer
    n = max(1, min(n, most // (rows * d)))
    case = {"op": op, "n": n, "rows": rows, "d": d, "type": kind, "bias": rng.random() < 0.5}
    if op == "train":
        case["weighted"] = rng.random() < 0.5
    return case


def _popular(gen, n, rows):
    """n ids, popular ones more often (Zipf-Mandelbrot, as rating sets are), in a shuffled numbering."""
    weight = (torch.arange(rows, device="cuda", dtype=torch.float64) + 21.0) ** -1.0
    cdf = torch.cumsum(weight / weight.sum(), 0)
    names = torch.randperm(rows, device="cuda", generator=gen)
    at = torch.searchsorted(cdf, torch.rand(n, device="cuda", dtype=torch.float64, generator=gen)).clamp_(max=rows - 1)
    return names[at].int()


def _pieces(case):
    """Shapes of the gradients: the user table in `pieces` unequal parts, the item table, both biases."""
    rows, cols, d, k = case["rows"], case["cols"], case["d"], case["pieces"]
    k = min(k, rows)
    edges = [rows * i * (i + 1) // (k * (k + 1)) for i in range(k + 1)]
    return [(b - a, d) for a, b in zip(edges, edges[1:])] + [(cols, d), (rows,), (cols,)]


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, op = _TYPES[case["type"]], case["op"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if op == "clip":
        grads = [(normal(*s) * 0.01).to(kind) for s in _pieces(case)]
        n = sum(g.numel() for g in grads)
        # the norm lies near 0.01 sqrt(n): a bound well under it, or over it
        return {"grads": grads, "most": (0.3 if case["clipped"] else 3.0) * 0.01 * n ** 0.5}
    n, rows, d = case["n"], case["rows"], case["d"]
    ids = _popular(gen, n, rows)
    # a twentieth of a batch is padding
    ids = torch.where(torch.rand(n, device="cuda", generator=gen) < 0.05, torch.full_like(ids, -1), ids)
    if op == "lookup":
        return {"table": (normal(rows, d) / d ** 0.5).to(kind), "ids": ids, "scale": d ** 0.5}
    if op == "lookup_grad":
        return {"grad": (normal(n, d) * 0.1).to(kind), "ids": ids, "rows": rows, "scale": d ** 0.5}
    if n == 1:
        ids = ids.clamp(min=0)
    # logits with a standard deviation of about 2, log-popularity as the items' bias
    inputs = {"x": normal(n, d).to(kind), "table": (normal(rows, d) * 2 / d ** 0.5).to(kind), "targets": ids, "bias": None, "scale": 1.0}
    if case["bias"]:
        inputs["bias"] = normal(rows)
    if op == "train":
        inputs["weights"] = torch.rand(n, device="cuda", generator=gen) / n if case["weighted"] else 1.0 / n
    return inputs


def prepare(case, seed):
    state = _inputs(case, seed)
    state["op"] = case["op"]
    if case["op"] == "clip":
        state["out"] = [torch.empty_like(g) for g in state["grads"]]
    return state


def _plain_loss(state):
    x, table, targets = state["x"].float(), state["table"].float(), state["targets"].long()
    z = torch.matmul(x, table.t()) * state["scale"]
    if state["bias"] is not None:
        z = z + state["bias"]
    top = z.amax(1, keepdim=True)
    lse = top[:, 0] + torch.log(torch.exp(z - top).sum(1))
    there = targets >= 0                # padding is left out: its loss and its log-sum are 0
    at = targets.clamp(min=0)[:, None]
    loss = torch.where(there, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse))
    return z, lse, loss, there, at


def run(state):
    op = state["op"]
    if own:
        import recommender_amd as ra
        if op == "lookup":
            return ra.embedding(state["table"], state["ids"], scale=state["scale"])
        if op == "lookup_grad":
            return ra.embedding_grad(state["grad"], state["ids"], state["rows"], scale=state["scale"])
        if op == "loss":
            return ra.softmax_loss(state["x"], state["table"], state["targets"], bias=state["bias"], scale=state["scale"])
        if op == "train":
            return ra.softmax_loss_grads(state["x"], state["table"], state["targets"], bias=state["bias"], scale=state["scale"],
                                         weights=state["weights"])
        norm = ra.clip_grads(state["grads"], state["most"], out=state["out"])
        return [norm] + state["out"]
    if op == "lookup":
        ids = state["ids"].long()
        rows = state["table"][ids.clamp(min=0)].float() * state["scale"]
        return (rows * (ids >= 0)[:, None]).to(state["table"].dtype)
    if op == "lookup_grad":
        ids = state["ids"].long()
        sums = torch.zeros(state["rows"] + 1, state["grad"].shape[1], device="cuda")       # padding goes to the last row
        sums.index_add_(0, torch.where(ids >= 0, ids, torch.full_like(ids, state["rows"])), state["grad"].float())
        return (sums[:-1] * state["scale"]).to(state["grad"].dtype)
    if op == "loss":
        _, lse, loss, there, _ = _plain_loss(state)
        return loss, lse * there
    if op == "train":
        z, lse, loss, there, at = _plain_loss(state)
        weights = there * state["weights"]
        g = torch.exp(z - lse[:, None])
        g.scatter_add_(1, at, torch.full_like(g[:, :1], -1.0))
        g = g * weights[:, None]
        dx = torch.matmul(g, state["table"].float()) * state["scale"]
        dtable = torch.matmul(g.t(), state["x"].float()) * state["scale"]
        dbias = None if state["bias"] is None else g.sum(0)
        return loss, lse * there, dx.to(state["x"].dtype), dtable.to(state["table"].dtype), dbias
    norm = torch.stack([(g.float() * g.float()).sum() for g in state["grads"]]).sum().sqrt()
    factor = torch.clamp(state["most"] / norm, max=1.0)
    return [norm] + [(g.float() * factor).to(g.dtype) for g in state["grads"]]


def work(case):
    size = 4 if case["type"] == "f32" else 2
    op = case["op"]
    if op == "clip":
        n = sum(s[0] * (s[1] if len(s) > 1 else 1) for s in _pieces(case))
        return {"bytes": 2 * n * size, "flops": 3 * n}
    n, rows, d = case["n"], case["rows"], case["d"]
    if op == "lookup":
        return {"bytes": 4 * n + (n + min(n, rows)) * d * size, "flops": n * d}
    if op == "lookup_grad":
        return {"bytes": 4 * n + (n + rows) * d * size, "flops": n * d}
    small = 12 * n + (4 * rows if case["bias"] else 0)
    if op == "loss":
        return {"bytes": (n + rows) * d * size + small, "flops": 2 * n * d * rows}
    return {"bytes": 2 * (n + rows) * d * size + 2 * small, "flops": 6 * n * d * rows}


def exact(case, seed):
    """The operators' definitions in 64 bits, a stretch of rows at a time."""
    given, op = _inputs(case, seed), case["op"]
    if op == "clip":
        norm = sum(float((g.double() ** 2).sum()) for g in given["grads"]) ** 0.5
        cut = min(1.0, given["most"] / norm)
        return [torch.tensor(norm, dtype=torch.float64)] + [g.double() * cut for g in given["grads"]]
    if op == "lookup":
        found = torch.zeros(case["n"], case["d"], dtype=torch.float64, device="cuda")
        live = torch.nonzero(given["ids"] >= 0)[:, 0]
        found[live] = given["table"][given["ids"][live].long()].double() * given["scale"]
        return found
    if op == "lookup_grad":
        # sums of equal ids as differences of running sums lose bits; a sorted segment sum does not
        live = torch.nonzero(given["ids"] >= 0)[:, 0]
        found = torch.zeros(case["rows"], case["d"], dtype=torch.float64, device="cuda")
        found.index_put_((given["ids"][live].long(),), given["grad"][live].double() * given["scale"], accumulate=True)
        return found
    x, w, t = given["x"].double(), given["table"].double(), given["targets"].long()
    n, rows = case["n"], case["rows"]
    loss, lse = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    db = torch.zeros(rows, dtype=torch.float64, device="cuda")
    many = max(1, (1 << 28) // rows)
    for a in range(0, n, many):
        z = given["scale"] * (x[a:a + many] @ w.T)
        if given["bias"] is not None:
            z += given["bias"].double()
        live = torch.nonzero(t[a:a + many] >= 0)[:, 0]
        lse[a + live] = torch.logsumexp(z, 1)[live]
        hit = t[a:a + many][live]
        loss[a + live] = lse[a + live] - z[live, hit]
        if op == "train":
            z = torch.softmax(z, 1)
            z[live, hit] -= 1.0
            share = torch.zeros(z.shape[0], dtype=torch.float64, device="cuda")
            g = given["weights"]
            share[live] = g[a + live].double() if torch.is_tensor(g) else g
            z *= share[:, None]
            dx[a:a + many] = given["scale"] * (z @ w)
            dw += given["scale"] * (z.T @ x[a:a + many])
            db += z.sum(0)
    if op == "loss":
        return loss, lse
    return loss, lse, dx, dw, db if given["bias"] is not None else None
