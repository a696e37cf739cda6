"""What is timed of the language-model operators in esgd.ops, with each operator's plain form.

Three families, as a training step of a language model meets them around its matrix products,
each with the gradients that the optimizer's buckets then carry:

  embedding   rows of a table looked up by token and scaled; the table's gradient, the sum of
              the output's gradient rows by token (tokens outside the table read zeros and
              give no gradient)
  experts     the (token, choice) pairs of a router sorted by expert, the tokens' rows copied
              to that order, the experts' rows brought back with their weights, and the
              gradients of both
  distill     the loss of a student's logits against a teacher's top logits at a temperature,
              per row, and its gradient in the student's logits

`own` chooses the side: False computes the formulas with elementary torch operations in 32 bits
(64 for the table gradient's sums, which may run over thousands of rows), True calls esgd.ops.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _ops():
    here = os.path.join(os.getcwd(), "eager-sgd_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    from esgd import ops
    return ops


# ---- cases ---------------------------------------------------------------------------------

def listed():
    return [
        # a few new tokens at once, as a server looks them up: latency only
        dict(name="lookup_few", op="lookup", tokens=16, rows=32768, width=1024, table="bf16", out="bf16",
             skew=2.0, pad=0.0, scale=32.0),
        # a long prompt from fp32 master weights into bf16 activations
        dict(name="lookup_prompt", op="lookup", tokens=8192, rows=131072, width=2048, table="f32", out="bf16",
             skew=2.0, pad=0.0, scale=1.0),
        # a small model's training step, every size odd: rows start off every alignment but the element's
        dict(name="embedding_odd", op="embedding", tokens=4095, rows=30011, width=1001, table="f32", out="f32",
             skew=1.0, pad=0.1, scale=0.5),
        # a training step's table: bf16 activations, an fp32 gradient bucket of 512 MiB, frequent tokens
        dict(name="embedding_large", op="embedding", tokens=32768, rows=131072, width=1024, table="f32", out="bf16",
             skew=3.0, pad=0.05, scale=32.0),
        # a few tokens through a small router while serving
        dict(name="experts_few", op="experts", tokens=16, choices=2, experts=8, width=1024, dtype="bf16",
             drop=0.0, train=False),
        # the order alone, for many tokens and experts: whole numbers only
        dict(name="experts_sort", op="sort", tokens=65536, choices=8, experts=256, drop=0.05),
        # a training step with odd sizes and dropped choices, fp32
        dict(name="experts_odd", op="experts", tokens=4095, choices=3, experts=61, width=769, dtype="f32",
             drop=0.1, train=True),
        # a large training step: 512 MiB of dispatched rows
        dict(name="experts_large", op="experts", tokens=16384, choices=8, experts=128, width=2048, dtype="bf16",
             drop=0.0, train=True),
        # a classifier's step: 64 images, 1001 classes, as the ResNet-50 example trains
        dict(name="distill_classes", op="distill", rows=64, vocab=1001, pitch=1001, top=10, dtype="f32",
             temperature=4.0, empty=0.0, invalid=0.0, train=True),
        # the loss alone on a few rows of a long vocabulary: one row's length has to be shared
        dict(name="distill_few", op="distill", rows=8, vocab=131072, pitch=131072, top=64, dtype="bf16",
             temperature=1.0, empty=0.0, invalid=0.0, train=False),
        # a training step on an odd vocabulary in a padded buffer, with rows that have no teacher
        dict(name="distill_odd", op="distill", rows=1023, vocab=49999, pitch=50048, top=100, dtype="f16",
             temperature=2.0, empty=0.1, invalid=0.1, train=True),
        # a large training step: 2 GiB of logits and as much gradient
        dict(name="distill_large", op="distill", rows=8192, vocab=131072, pitch=131072, top=64, dtype="bf16",
             temperature=1.0, empty=0.02, invalid=0.0, train=True),
    ]


def _between(rng, low, high):
    """A size from low to high, spread over its logarithm, odd as often as not."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["lookup", "embedding", "experts", "sort", "distill", "distill"])
    kind = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op in ("lookup", "embedding"):
        rows, width = _between(rng, 512, 131072), _between(rng, 32, 2048)
        table = rng.choice(["f32", kind])
        return dict(op=op, tokens=_between(rng, 1, 32768), rows=rows, width=min(width, 131072 * 1024 // rows), table=table,
                    out=kind if table == "f32" else table, skew=rng.choice([1.0, 2.0, 3.0]),
                    pad=rng.choice([0.0, 0.05, 0.3]), scale=rng.choice([1.0, 0.5, 32.0]))
    if op in ("experts", "sort"):
        choices = rng.randint(1, 8)
        tokens = _between(rng, 1, 16384)
        case = dict(op=op, tokens=tokens, choices=choices, experts=_between(rng, 2, 512), drop=rng.choice([0.0, 0.1]))
        if op == "sort":
            return dict(case, tokens=4 * tokens)
        return dict(case, width=_between(rng, 32, 1024 if kind == "f32" else 2048), dtype=kind, train=rng.random() < 0.7)
    vocab = _between(rng, 500, 131072)
    most = (1 << 29) // vocab
    return dict(op="distill", rows=_between(rng, 1, min(8192, most)), vocab=vocab, pitch=vocab + rng.choice([0, 0, 1, 64]),
                top=rng.randint(1, 128), dtype=kind, temperature=rng.choice([1.0, 2.0, 4.0]), empty=rng.choice([0.0, 0.1]),
                invalid=rng.choice([0.0, 0.1]), train=rng.random() < 0.8)


# ---- inputs --------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype, scale=1.0):
        return torch.randn(*shape, device=dev, generator=g).mul_(scale).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, device=dev, generator=g)

    s = dict(case=case)
    if case["op"] in ("lookup", "embedding"):
        # token numbers by falling frequency, some of them the padding's -1
        t = (uniform(case["tokens"]).double().pow(case["skew"]) * case["rows"]).long().clamp_(max=case["rows"] - 1)
        t = torch.where(uniform(case["tokens"]) < case["pad"], torch.full_like(t, -1), t)
        s["tokens"] = t
        s["weight"] = normal(case["rows"], case["width"], dtype=DTYPES[case["table"]], scale=0.02)
        if case["op"] == "embedding":
            s["grad"] = normal(case["tokens"], case["width"], dtype=DTYPES[case["out"]])
        return s
    if case["op"] in ("experts", "sort"):
        n, k, e = case["tokens"], case["choices"], case["experts"]
        # some experts are more wanted than others; a dropped choice names none
        pick = (uniform(n, k).pow(1.5) * e).to(torch.int32).clamp_(max=e - 1)
        s["pick"] = torch.where(uniform(n, k) < case["drop"], torch.full_like(pick, -1), pick)
        if case["op"] == "experts":
            dt, d = DTYPES[case["dtype"]], case["width"]
            s["weights"] = torch.softmax(torch.randn(n, k, device=dev, generator=g), dim=-1)
            s["x"] = normal(n, d, dtype=dt)
            s["y"] = normal(n * k, d, dtype=dt)   # what the experts made of the dispatched rows
            if case["train"]:
                s["grad_rows"] = normal(n * k, d, dtype=dt)
                s["grad_out"] = normal(n, d, dtype=dt)
        return s
    n, v, k = case["rows"], case["vocab"], case["top"]
    k = min(k, v)
    part = v // k
    index = torch.arange(k, device=dev) * part + (uniform(n, k) * part).long().clamp_(max=part - 1)
    index = (index + (uniform(n, 1) * v).long()) % v
    top = (uniform(n, k) * 8.0).sort(dim=-1, descending=True).values
    z = torch.empty(n, case["pitch"], device=dev, dtype=DTYPES[case["dtype"]])
    step = max(1, (1 << 28) // case["pitch"])
    for a in range(0, n, step):   # the student has learnt a part of what the teacher says
        part_z = torch.randn(min(step, n - a), case["pitch"], device=dev, generator=g)
        part_z.scatter_add_(1, index[a:a + step], top[a:a + step] * 0.7)
        z[a:a + step] = part_z
    s["logits"] = z[:, :v]
    index = torch.where(uniform(n, k) < case["invalid"], torch.full_like(index, -1), index)
    s["top_index"] = torch.where(uniform(n, 1) < case["empty"], torch.full_like(index, -1), index)
    s["top_logits"] = top.to(DTYPES[case["dtype"]])
    # the mean's gradient, times a loss scale where 16 bits have few exponents
    s["row_grad"] = torch.full((n,), (4096.0 if case["dtype"] == "f16" else 1.0) / n, device=dev)
    return s


# ---- one pass ------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if case["op"] == "lookup":
        return {"out": _lookup(s)}
    if case["op"] == "embedding":
        return {"out": _lookup(s), "grad_weight": _table_gradient(s)}
    if case["op"] == "sort":
        offsets, slots, _ = _order(s)
        return {"offsets": offsets, "slots": slots}
    if case["op"] == "experts":
        return _experts(s)
    return _distill(s)


def _lookup(s):
    case = s["case"]
    if own:
        return _ops().embedding(s["weight"], s["tokens"], case["scale"], dtype=DTYPES[case["out"]])
    t = s["tokens"]
    known = (t >= 0) & (t < case["rows"])
    rows = s["weight"][t.clamp(0, case["rows"] - 1)].float() * case["scale"]
    return torch.where(known[:, None], rows, torch.zeros_like(rows)).to(DTYPES[case["out"]])


def _table_gradient(s):
    case = s["case"]
    if own:
        return _ops().embedding_grad(s["grad"], s["tokens"], case["rows"], case["scale"], dtype=DTYPES[case["table"]])
    t = s["tokens"]
    known = (t >= 0) & (t < case["rows"])
    grad = torch.where(known[:, None], s["grad"], torch.zeros_like(s["grad"])).double()
    table = torch.zeros(case["rows"], case["width"], device=t.device, dtype=torch.float64)
    table.index_add_(0, t.clamp(0, case["rows"] - 1), grad)
    return (table * case["scale"]).to(DTYPES[case["table"]])


def _order(s):
    """(offsets, slots, what the framework keeps): slots[t, j] is where choice j of token t stands in
    the order by expert, equal experts by (t, j); a dropped choice's place p behind them is -1 - p."""
    case = s["case"]
    if own:
        order = _ops().expert_sort(s["pick"], case["experts"])
        return order.offsets, order.slots, order
    flat = s["pick"].reshape(-1)
    dropped = (flat < 0) | (flat >= case["experts"])
    key = torch.where(dropped, torch.full_like(flat, case["experts"]), flat)
    by_expert = torch.argsort(key, stable=True)
    place = torch.empty_like(by_expert)
    place[by_expert] = torch.arange(flat.numel(), device=flat.device)
    slots = torch.where(dropped, -1 - place, place).to(torch.int32).view_as(s["pick"])
    ends = torch.cumsum(torch.bincount(key, minlength=case["experts"] + 1)[:case["experts"]], 0)
    offsets = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    return offsets, slots, None


def _experts(s):
    case = s["case"]
    offsets, slots, order = _order(s)
    got = {"offsets": offsets, "slots": slots}
    if own:
        ops = _ops()
        got["rows"] = ops.expert_dispatch(s["x"], order)
        got["out"] = ops.expert_combine(s["y"], s["weights"], order)
        if case["train"]:
            got["grad_y"], got["grad_weights"] = ops.expert_combine_grad(s["grad_out"], s["y"], s["weights"], order)
            got["grad_x"] = ops.expert_dispatch_grad(s["grad_rows"], order)
        return got
    n, k, dt = case["tokens"], case["choices"], DTYPES[case["dtype"]]
    kept = slots >= 0
    place = torch.where(kept, slots, -1 - slots).long()
    rows = torch.empty(n * k, case["width"], device=slots.device, dtype=dt)
    rows[place.reshape(-1)] = torch.where(kept[..., None], s["x"][:, None, :], torch.zeros_like(s["x"])[:, None, :]).reshape(n * k, -1)
    got["rows"] = rows
    w = torch.where(kept, s["weights"], torch.zeros_like(s["weights"]))
    y = torch.where(kept[..., None], s["y"][place].float(), torch.zeros((), device=slots.device))
    got["out"] = (w[..., None] * y).sum(1).to(dt)
    if case["train"]:
        g = s["grad_out"].float()
        grad_y = torch.empty_like(rows)
        grad_y[place.reshape(-1)] = (w[..., None] * g[:, None, :]).to(dt).reshape(n * k, -1)
        got["grad_y"] = grad_y
        got["grad_weights"] = (y * g[:, None, :]).sum(-1)
        gr = torch.where(kept[..., None], s["grad_rows"][place].float(), torch.zeros((), device=slots.device))
        got["grad_x"] = gr.sum(1).to(dt)
    return got


def _distill(s):
    case = s["case"]
    tau = case["temperature"]
    if own:
        if not case["train"]:
            return {"loss": _ops().distill_loss(s["logits"], s["top_logits"], s["top_index"], tau)}
        loss, grad = _ops().distill_loss_grad(s["logits"], s["top_logits"], s["top_index"], s["row_grad"], tau)
        return {"loss": loss, "grad_logits": grad}
    z = s["logits"].float() / tau
    known = (s["top_index"] >= 0) & (s["top_index"] < case["vocab"])
    at = s["top_index"].clamp(0, case["vocab"] - 1)
    t = torch.where(known, s["top_logits"].float() / tau, torch.full((), -math.inf, device=z.device))
    t_max = t.max(-1, keepdim=True).values
    some = t_max > -math.inf
    e = torch.exp(t - torch.where(some, t_max, torch.zeros_like(t_max)))
    total = torch.where(some, e.sum(-1, keepdim=True), torch.ones_like(t_max))
    p = e / total
    log_p = t - torch.where(some, t_max, torch.zeros_like(t_max)) - torch.log(total)
    z_max = z.max(-1, keepdim=True).values
    ez = torch.exp(z - z_max)
    ez_sum = ez.sum(-1, keepdim=True)
    log_q = z.gather(1, at) - z_max - torch.log(ez_sum)
    loss = torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(-1) * (tau * tau)
    loss = torch.where(some[:, 0], loss, torch.zeros_like(loss))
    if not case["train"]:
        return {"loss": loss}
    scale = torch.where(some, s["row_grad"][:, None] * tau, torch.zeros_like(t_max))
    grad = ez * (scale / ez_sum)
    grad.scatter_add_(1, at, -p * scale)
    return {"loss": loss, "grad_logits": grad.to(DTYPES[case["dtype"]])}


# ---- what a pass cannot do without ---------------------------------------------------------

def _different_tokens(case):
    """How many rows of the table the tokens name, as expected of their distribution."""
    edges = torch.arange(case["rows"] + 1, dtype=torch.float64).div_(case["rows"]).pow_(1.0 / case["skew"])
    p = edges[1:] - edges[:-1]
    return float((1 - torch.exp(case["tokens"] * (1 - case["pad"]) * torch.log1p(-p.clamp(max=1 - 1e-15)))).sum())


def work(case):
    if case["op"] in ("lookup", "embedding"):
        n, d = case["tokens"], case["width"]
        moved = 8 * n + _different_tokens(case) * d * BYTES[case["table"]] + n * d * BYTES[case["out"]]
        flops = n * d
        if case["op"] == "embedding":
            moved += n * (1 - case["pad"]) * d * BYTES[case["out"]] + case["rows"] * d * BYTES[case["table"]]
            flops += 2 * n * d
        return {"bytes": moved, "flops": flops}
    if case["op"] in ("experts", "sort"):
        n, k = case["tokens"], case["choices"]
        moved, flops = 8 * n * k + 4 * (case["experts"] + 1), 0
        if case["op"] == "experts":
            one, kept = case["width"] * BYTES[case["dtype"]], n * k * (1 - case["drop"])
            moved += n * one + n * k * one                       # x read, its rows written
            moved += kept * one + n * one + 4 * n * k            # the experts' rows read, the sum written
            flops += 2 * kept * case["width"]
            if case["train"]:
                moved += n * one + n * k * one + 4 * n * k       # the sum's gradient read; grad_y and grad_weights written
                moved += kept * one + n * one                    # the rows' gradient read, x's written
                flops += 4 * kept * case["width"]
        return {"bytes": moved, "flops": flops}
    n, v, b = case["rows"], case["vocab"], BYTES[case["dtype"]]
    moved = n * v * b * (2 if case["train"] else 1) + n * min(case["top"], v) * (8 + b) + 4 * n * (2 if case["train"] else 1)
    return {"bytes": moved, "flops": n * v * (6 if case["train"] else 3)}


# ---- the definition in 64 bits -------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sort":
        return None
    if case["op"] in ("lookup", "embedding"):
        t = s["tokens"]
        inside = torch.nonzero((t >= 0) & (t < case["rows"]))[:, 0]
        out = torch.zeros(t.numel(), case["width"], dtype=torch.float64, device=t.device)
        out[inside] = s["weight"].index_select(0, t[inside]).double() * case["scale"]
        if case["op"] == "lookup":
            return {"out": out}
        # the gradient rows in the tokens' order, summed from the first: a token's rows lie together
        table = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device=t.device)
        if inside.numel():
            names, at = torch.sort(t[inside])
            run_of, counts = torch.unique_consecutive(names, return_counts=True)
            ends = counts.cumsum(0) - 1
            sums = s["grad"][inside[at]].double().cumsum(0)[ends]
            table[run_of] = torch.diff(sums, dim=0, prepend=torch.zeros_like(sums[:1])) * case["scale"]
        return {"out": out, "grad_weight": table}
    if case["op"] == "experts":
        n, k = case["tokens"], case["choices"]
        flat = s["pick"].reshape(-1).long()
        pairs = torch.cat([torch.nonzero(flat == e)[:, 0] for e in range(case["experts"])])   # kept ones, by expert
        token = pairs // k
        w = s["weights"].double().reshape(-1)[pairs, None]
        m = pairs.numel()
        rows = torch.zeros(n * k, case["width"], dtype=torch.float64, device=flat.device)
        rows[:m] = s["x"].double()[token]
        out = torch.zeros(n, case["width"], dtype=torch.float64, device=flat.device)
        out.index_add_(0, token, w * s["y"][:m].double())
        got = {"offsets": None, "slots": None, "rows": rows, "out": out}
        if case["train"]:
            g = s["grad_out"].double()[token]
            got["grad_y"] = torch.zeros_like(rows)
            got["grad_y"][:m] = w * g
            got["grad_weights"] = torch.zeros(n * k, dtype=torch.float64, device=flat.device)
            got["grad_weights"][pairs] = (g * s["y"][:m].double()).sum(1)
            got["grad_weights"] = got["grad_weights"].view(n, k)
            got["grad_x"] = torch.zeros_like(out).index_add_(0, token, s["grad_rows"][:m].double())
        return got
    tau, v = case["temperature"], case["vocab"]
    n = case["rows"]
    loss = torch.zeros(n, dtype=torch.float64, device=s["logits"].device)
    grad = torch.zeros(n, v, dtype=torch.float64, device=loss.device) if case["train"] else None
    step = max(1, (1 << 27) // v)
    for a in range(0, n, step):
        z = s["logits"][a:a + step].double() / tau
        index = s["top_index"][a:a + step]
        known = (index >= 0) & (index < v)
        said = (s["top_logits"][a:a + step].double() / tau).masked_fill(~known, -math.inf)
        with_teacher = torch.nonzero(known.any(1))[:, 0]
        if not with_teacher.numel():
            continue
        z, index, said, known = z[with_teacher], index[with_teacher], said[with_teacher], known[with_teacher]
        log_p = torch.log_softmax(said, -1)
        p = log_p.exp()
        log_q = torch.log_softmax(z, -1)
        terms = p * (log_p - log_q.gather(1, index.clamp(min=0)))
        loss[a + with_teacher] = terms.masked_fill(~known, 0.0).sum(1) * tau ** 2
        if grad is not None:
            d = log_q.exp_()
            d.scatter_add_(1, index.clamp(min=0), -p)
            grad[a + with_teacher] = d * (s["row_grad"][a + with_teacher].double() * tau)[:, None]
    return {"loss": loss, "grad_logits": grad} if case["train"] else {"loss": loss}
