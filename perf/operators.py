"""Cases of the per-row-id operators: sorting rows by id, embedding lookup with its gradient, products with the
weights of a row's group, and distillation from a teacher's top logits.

``run`` computes a case in elementary torch operations where ``own`` is false and through the framework's entry
points where it is true; ``exact`` computes it from the definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # 64 tokens routed to 8 groups: the sort of a serving step, latency only
        {"name": "group-64", "op": "group", "n": 64, "groups": 8, "outside": 0.0},
        # a million ids over a vocabulary, log-uniform as token frequencies are, a few of them padding
        {"name": "group-1m", "op": "group", "n": 1000003, "groups": 50021, "outside": 0.02},
        # one token's embedding row, the lookup of a decoding step
        {"name": "embed-1", "op": "embed", "n": 1, "rows": 50021, "width": 1024, "dtype": "bf16", "train": False,
         "scale": 32.0, "outside": 0.0},
        # a class embedding (512 wide, 36 classes) for each voxel of a batch, unlabelled voxels at -1; training
        {"name": "embed-classes", "op": "embed", "n": 92001, "rows": 36, "width": 512, "dtype": "fp32", "train": True,
         "scale": 1.0, "outside": 0.1},
        # a training step's tokens over a vocabulary
        {"name": "embed-vocab", "op": "embed", "n": 32768, "rows": 65536, "width": 1024, "dtype": "bf16", "train": True,
         "scale": 32.0, "outside": 0.0},
        # eight tokens of a serving step over 16 groups' weights
        {"name": "linear-8", "op": "linear", "n": 8, "groups": 16, "in": 1024, "out": 2048, "dtype": "bf16", "bias": False,
         "train": False, "outside": 0.0},
        # an odd, ragged, biased forward pass; some rows belong to no group
        {"name": "linear-odd", "op": "linear", "n": 5003, "groups": 7, "in": 203, "out": 131, "dtype": "fp16", "bias": True,
         "train": False, "outside": 0.05},
        # the 96 -> 512 projection head with weights of its own for each of three datasets; training
        {"name": "linear-heads", "op": "linear", "n": 92417, "groups": 3, "in": 96, "out": 512, "dtype": "fp32",
         "bias": True, "train": True, "outside": 0.0},
        # 16 experts' products, training
        {"name": "linear-experts", "op": "linear", "n": 32768, "groups": 16, "in": 1024, "out": 1024, "dtype": "bf16",
         "bias": False, "train": True, "outside": 0.0},
        # one row of a large vocabulary
        {"name": "distil-1", "op": "distil", "n": 1, "classes": 131072, "top": 16, "dtype": "fp32", "temperature": 2.0,
         "blank": 0.0},
        # 25 valid classes for each voxel of a batch
        {"name": "distil-classes", "op": "distil", "n": 92001, "classes": 25, "top": 5, "dtype": "fp32",
         "temperature": 1.0, "blank": 0.1},
        # a training step over a vocabulary of odd size
        {"name": "distil-vocab", "op": "distil", "n": 4096, "classes": 65537, "top": 32, "dtype": "bf16",
         "temperature": 2.0, "blank": 0.02},
    ]


def _spread(rng, low, high):
    """A whole number, spread over the logarithm of low .. high."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["group", "embed", "linear", "distil"])
    dtype = rng.choice(sorted(DTYPES))

    def some(n):  # the share of rows without an id or a list, none of them where there are few
        return rng.choice([0.0, 0.02, 0.1]) if n >= 64 else 0.0

    if op == "group":
        n = _spread(rng, 16, 1000003)
        return {"op": op, "n": n, "groups": _spread(rng, 2, 65536), "outside": some(n)}
    if op == "embed":
        rows, width = _spread(rng, 13, 65536), _spread(rng, 8, 1024)
        n = _spread(rng, 1, min(131072, 32768 * 1024 // width))
        return {"op": op, "n": n, "rows": rows, "width": width, "dtype": dtype, "train": rng.random() < 0.6,
                "scale": rng.choice([1.0, math.sqrt(width)]), "outside": some(n)}
    if op == "linear":
        k, n = _spread(rng, 16, 2048), _spread(rng, 16, 2048)
        most = 32768 * 1024 * 1024 // (k * n * (4 if dtype == "fp32" else 1))
        rows = _spread(rng, 1, max(1, min(131072, most)))
        return {"op": op, "n": rows, "groups": _spread(rng, 1, 64), "in": k, "out": n, "dtype": dtype,
                "bias": rng.random() < 0.5, "train": rng.random() < 0.6, "outside": some(rows)}
    classes = _spread(rng, 13, 131072)
    most = 4096 * 65536 // (classes * (2 if dtype == "fp32" else 1))
    n = _spread(rng, 1, max(1, min(131072, most)))
    return {"op": op, "n": n, "classes": classes, "top": min(classes, _spread(rng, 1, 64)), "dtype": dtype,
            "temperature": rng.choice([1.0, 2.0, 4.0]), "blank": some(n)}


# ------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ids(n, count, outside, g):
    """n ids of 0 .. count - 1, log-uniform as token frequencies are, a share of them -1."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(count + 1.0)) - 1.0).long().clamp_(0, count - 1)
    return torch.where(torch.rand(n, generator=g, device="cuda") < outside, torch.full_like(ids, -1), ids)


def _routed(n, groups, outside, g):
    """n ids of 0 .. groups - 1, the groups' shares within a factor of two of each other, a share of the ids -1."""
    share = 1.0 + torch.rand(groups, generator=g, device="cuda")
    ids = torch.multinomial(share, n, replacement=True, generator=g)
    return torch.where(torch.rand(n, generator=g, device="cuda") < outside, torch.full_like(ids, -1), ids)


def prepare(case, seed):
    g, op, n = _generator(seed), case["op"], case["n"]
    s = dict(case)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(DTYPES[case["dtype"]])

    if op == "group":
        s["index"] = _ids(n, case["groups"], case["outside"], g)
    elif op == "embed":
        s["index"] = _ids(n, case["rows"], case["outside"], g)
        s["weight"] = normal(case["rows"], case["width"], std=0.02)
        if case["train"]:
            s["grad"] = normal(n, case["width"])
    elif op == "linear":
        s["index"] = _routed(n, case["groups"], case["outside"], g)
        s["longest"] = max(1, int(torch.bincount(s["index"].clamp(min=0), minlength=1).max()))
        s["x"] = normal(n, case["in"])
        s["weight"] = normal(case["groups"], case["out"], case["in"], std=case["in"] ** -0.5)
        s["bias"] = normal(case["groups"], case["out"], std=0.1) if case["bias"] else None
        if case["train"]:
            s["grad"] = normal(n, case["out"])
    else:
        v, k = case["classes"], case["top"]
        top = torch.randint(0, v, (n, k), generator=g, device="cuda")
        s["teacher_logits"] = torch.randn((n, k), generator=g, device="cuda").mul_(3.0).sort(1, descending=True).values
        logits = normal(n, v, std=2.0)
        # the student agrees with the teacher's first choice about half of the time
        half = torch.rand((n, 1), generator=g, device="cuda") < 0.5
        s["logits"] = logits.scatter_add_(1, top[:, :1], (half * 6.0).to(logits.dtype))
        # lists shorter than k end in -1; a share of the rows has no list at all
        length = k - torch.randint(0, 1 + k // 4, (n, 1), generator=g, device="cuda")
        length = torch.where(torch.rand((n, 1), generator=g, device="cuda") < case["blank"],
                             torch.zeros_like(length), length)
        s["teacher_index"] = torch.where(torch.arange(k, device="cuda") < length, top, torch.full_like(top, -1))
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    return (_framework if own else _plain)[s["op"]](s)


def _plain_order(index, count):
    """The stable order of the rows by id (ids outside 0 .. count - 1 last) and the groups' offsets."""
    key = torch.where((index >= 0) & (index < count), index, torch.full_like(index, count))
    sizes = torch.zeros(count + 1, dtype=torch.long, device=index.device).scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cumsum(sizes, 0) - sizes
    return key, torch.sort(key, stable=True).indices, offsets


def _plain_group(s):
    _, order, offsets = _plain_order(s["index"], s["groups"])
    return {"order": order.int(), "offsets": offsets.int()}


def _plain_embed(s):
    index, weight = s["index"], s["weight"]
    inside = ((index >= 0) & (index < s["rows"]))[:, None]
    at = index.clamp(0, s["rows"] - 1)
    y = torch.where(inside, weight[at].float() * s["scale"], 0.0)
    out = {"y": y.to(weight.dtype)}
    if s["train"]:
        g = torch.where(inside, s["grad"].float(), 0.0)
        dw = torch.zeros(weight.shape, device="cuda").index_add_(0, at, g)
        out["d_weight"] = (dw * s["scale"]).to(weight.dtype)
    return out


def _plain_linear(s):
    """The groups' rows in a padded batch (groups, longest, .), and one batched product in 32 bits."""
    x, weight, groups, longest = s["x"], s["weight"].float(), s["groups"], s["longest"]
    key, order, offsets = _plain_order(s["index"], groups)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device="cuda")
    slot = torch.where(key < groups, key * longest + place - offsets[key], groups * longest)
    inside = (key < groups)[:, None]

    def pad(t):
        p = torch.zeros((groups * longest + 1, t.shape[1]), device="cuda")
        p[slot] = t.float()
        p[-1] = 0.0
        return p[:-1].view(groups, longest, t.shape[1])

    def rows(p):
        flat = p.reshape(groups * longest, p.shape[2])
        return torch.where(inside, flat[slot.clamp(max=groups * longest - 1)], 0.0)

    xp = pad(x)
    y = torch.bmm(xp, weight.transpose(1, 2).contiguous())
    if s["bias"] is not None:
        y = y + s["bias"].float()[:, None, :]
    out = {"y": rows(y).to(x.dtype)}
    if s["train"]:
        gp = pad(s["grad"])
        out["d_x"] = rows(torch.bmm(gp, weight)).to(x.dtype)
        out["d_weight"] = torch.bmm(gp.transpose(1, 2).contiguous(), xp).to(x.dtype)
        if s["bias"] is not None:
            out["d_bias"] = gp.sum(1).to(x.dtype)
    return out


def _plain_distil(s):
    t = s["temperature"]
    logits = s["logits"].float() / t
    listed_ = (s["teacher_index"] >= 0) & (s["teacher_index"] < s["classes"])
    at = s["teacher_index"].clamp(0, s["classes"] - 1)
    some = listed_.any(1)
    teacher = torch.where(listed_, s["teacher_logits"].float() / t, -torch.inf)
    teacher = torch.where(some[:, None], teacher, 0.0)
    log_p = torch.log_softmax(teacher, 1)
    p = torch.where(listed_, torch.exp(log_p), 0.0)
    log_q = logits - torch.logsumexp(logits, 1, keepdim=True)
    terms = torch.where(p > 0, p * (log_p - torch.gather(log_q, 1, at)), 0.0)
    count = some.sum().clamp(min=1)
    loss = torch.where(some, terms.sum(1), 0.0).sum() * (t * t) / count
    grad = torch.exp(log_q).scatter_add_(1, at, -p) * (t / count)
    return {"loss": loss, "d_logits": torch.where(some[:, None], grad, 0.0).to(s["logits"].dtype)}


_plain = {"group": _plain_group, "embed": _plain_embed, "linear": _plain_linear, "distil": _plain_distil}


def _own_group(s):
    from ponderv2_amd.row_groups import group_rows

    groups = group_rows(s["index"], s["groups"])
    return {"order": groups.order, "offsets": groups.offsets}


def _own_embed(s):
    from ponderv2_amd.embedding import embedding

    if not s["train"]:
        return {"y": embedding(s["index"], s["weight"], scale=s["scale"])}
    weight = s["weight"].detach().requires_grad_()
    y = embedding(s["index"], weight, scale=s["scale"])
    return {"y": y.detach(), "d_weight": torch.autograd.grad(y, weight, s["grad"])[0]}


def _own_linear(s):
    from ponderv2_amd.grouped_linear import grouped_linear
    from ponderv2_amd.row_groups import group_rows

    groups = group_rows(s["index"], s["groups"])
    if not s["train"]:
        return {"y": grouped_linear(s["x"], s["weight"], groups, s["bias"])}
    leaves = {"d_x": s["x"].detach().requires_grad_(), "d_weight": s["weight"].detach().requires_grad_()}
    if s["bias"] is not None:
        leaves["d_bias"] = s["bias"].detach().requires_grad_()
    y = grouped_linear(leaves["d_x"], leaves["d_weight"], groups, leaves.get("d_bias"))
    grads = torch.autograd.grad(y, list(leaves.values()), s["grad"])
    return {"y": y.detach(), **dict(zip(leaves, grads))}


def _own_distil(s):
    from ponderv2_amd.distillation import topk_distillation

    logits = s["logits"].detach().requires_grad_()
    loss = topk_distillation(logits, s["teacher_index"], s["teacher_logits"], temperature=s["temperature"])
    return {"loss": loss.detach(), "d_logits": torch.autograd.grad(loss, logits)[0]}


_framework = {"group": _own_group, "embed": _own_embed, "linear": _own_linear, "distil": _own_distil}


# ------------------------------------------------------------------------------------------ from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    op, n = case["op"], case["n"]
    if op == "group":
        return None  # whole numbers only
    if op == "embed":
        table = torch.cat([s["weight"].double() * case["scale"],
                           torch.zeros((1, case["width"]), dtype=torch.float64, device="cuda")])
        last = case["rows"]
        at = [i if 0 <= i < last else last for i in s["index"].tolist()]
        at = torch.tensor(at, device="cuda")
        out = {"y": table[at]}
        if case["train"]:
            sums = torch.zeros_like(table).index_put_((at,), s["grad"].double(), accumulate=True)
            out["d_weight"] = sums[:last] * case["scale"]
        return out
    if op == "linear":
        out = {"y": torch.zeros((n, case["out"]), dtype=torch.float64, device="cuda")}
        if case["train"]:
            out["d_x"] = torch.zeros((n, case["in"]), dtype=torch.float64, device="cuda")
            out["d_weight"] = torch.zeros(s["weight"].shape, dtype=torch.float64, device="cuda")
            if case["bias"]:
                out["d_bias"] = torch.zeros((case["groups"], case["out"]), dtype=torch.float64, device="cuda")
        for group in range(case["groups"]):
            mine = torch.nonzero(s["index"] == group)[:, 0]
            x, w = s["x"][mine].double(), s["weight"][group].double()
            out["y"][mine] = x @ w.T + (s["bias"][group].double() if case["bias"] else 0.0)
            if case["train"]:
                g = s["grad"][mine].double()
                out["d_x"][mine] = g @ w
                out["d_weight"][group] = g.T @ x
                if case["bias"]:
                    out["d_bias"][group] = g.sum(0)
        return out
    t, v = case["temperature"], case["classes"]
    has = s["teacher_index"] >= 0
    rows = has.sum(1) > 0
    count = max(1, int(rows.sum()))
    z = torch.exp((s["teacher_logits"].double() - s["teacher_logits"].double().amax(1, keepdim=True)) / t) * has
    p = z / z.sum(1, keepdim=True).clamp(min=1e-300)
    target = torch.zeros((n, v + 1), dtype=torch.float64, device="cuda")
    target.scatter_add_(1, torch.where(has, s["teacher_index"], torch.full_like(s["teacher_index"], v)), p)
    target = target[:, :v]
    e = s["logits"].double() / t
    e -= e.amax(1, keepdim=True)
    total = torch.exp(e).sum(1, keepdim=True)
    at = s["teacher_index"].clamp(min=0)
    log_p = torch.log(torch.where(has, p, torch.ones_like(p)))
    losses = (p * (log_p - torch.gather(e, 1, at) + torch.log(total))).sum(1)
    grad = (torch.exp(e).div_(total) - target).mul_(rows[:, None] * (t / count))
    return {"loss": losses.sum() * t * t / count, "d_logits": grad}


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def _distinct(n, count):
    """How many of ``count`` log-uniform ids n draws meet."""
    v = torch.arange(1, count + 1, dtype=torch.float64)
    share = torch.log1p(1.0 / v) / math.log(count + 1.0)
    return float((1.0 - torch.exp(n * torch.log1p(-share.clamp(max=1.0 - 1e-12)))).sum())


def work(case):
    op, n = case["op"], case["n"]
    if op == "group":
        return {"bytes": 8 * n + 4 * n + 4 * (case["groups"] + 1), "flops": 0}
    b = BYTES[case["dtype"]]
    if op == "embed":
        c = case["width"]
        moved = 8 * n + _distinct(n, case["rows"]) * c * b + n * c * b
        flops = n * c
        if case["train"]:
            moved += n * c * b + case["rows"] * c * b
            flops += n * c
        return {"bytes": moved, "flops": flops}
    if op == "linear":
        g, k, m = case["groups"], case["in"], case["out"]
        used = g * (1.0 - (1.0 - 1.0 / g) ** n)
        weights = used * (k + case["bias"]) * m * b
        moved, flops = 8 * n + weights + n * (k + m) * b, 2.0 * n * k * m
        if case["train"]:
            moved, flops = moved + n * (k + m) * b + g * (k + case["bias"]) * m * b, 3.0 * flops
        return {"bytes": moved, "flops": flops}
    v, k = case["classes"], case["top"]
    return {"bytes": 2 * n * v * b + n * k * 12, "flops": 8.0 * n * v}
