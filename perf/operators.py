"""The losses of a language model's training step, as measurable cases.

Three operators, each in its plain form (torch operations in 32 bits) and as the library's calls:

* ``head``: softmax cross entropy of a vocabulary head. ``x [rows, dim]`` and ``w [classes, dim]`` give
  logits ``x w^T``; ``labels`` are int32 class ids, a negative one leaves its row out. A training step
  returns the loss, each row's log-sum-exp and both gradients; an evaluation the loss and the rows' own.
* ``distill``: the divergence of a student's softmax from a teacher's top logits. ``x [rows, classes]``
  are the student's logits, ``teacher [rows, k]`` the teacher's at the classes ``ids [rows, k]`` (negative:
  no entry). A training step returns the loss, each row's log-sum-exp and the logits' gradient.
* ``router``: a mixture-of-experts router. Softmax over ``x [rows, experts]``, the ``k`` largest logits of
  each row (ties to the lowest index), their weights, how often each expert was chosen, the balance loss
  ``experts * sum_e f_e P_e`` and the gradient of the logits. ``keep`` is 0 at padding rows.

Data is fp32, the library's one type; labels, ids and counts are int32.
"""
import math

import torch

own = False
_started = False


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------
def listed():
    return [
        # a head as small as a test model's: a handful of launches
        {"name": "head_small", "op": "head", "rows": 64, "dim": 128, "classes": 1000, "train": True},
        # an image classifier's head over a large batch, 1000 classes
        {"name": "head_1000", "op": "head", "rows": 32768, "dim": 512, "classes": 1000, "train": True},
        # evaluation of a language model: the loss of every token, no gradient
        {"name": "head_eval", "op": "head", "rows": 4096, "dim": 1024, "classes": 32000, "train": False},
        # a ragged micro-batch, and a vocabulary and width that no tile divides
        {"name": "head_odd", "op": "head", "rows": 1023, "dim": 513, "classes": 30011, "train": True},
        # a training step over a large vocabulary
        {"name": "head_large", "op": "head", "rows": 4096, "dim": 2048, "classes": 131072, "train": True},
        # distillation of a small classifier
        {"name": "distill_small", "op": "distill", "rows": 32, "classes": 1000, "k": 8, "temperature": 1.0},
        # a ragged micro-batch against a teacher's top 50
        {"name": "distill_odd", "op": "distill", "rows": 1025, "classes": 30011, "k": 50, "temperature": 2.0},
        # a training step over a large vocabulary against a teacher's top 128
        {"name": "distill_large", "op": "distill", "rows": 4096, "classes": 131072, "k": 128, "temperature": 1.5},
        # the router of a small model's batch
        {"name": "router_small", "op": "router", "rows": 64, "experts": 8, "k": 2, "normalise": True},
        # a micro-batch over 64 experts
        {"name": "router_64", "op": "router", "rows": 8192, "experts": 64, "k": 6, "normalise": False},
        # a ragged batch over a number of experts that is no power of two
        {"name": "router_odd", "op": "router", "rows": 33333, "experts": 60, "k": 5, "normalise": True},
        # a large batch over many experts
        {"name": "router_256", "op": "router", "rows": 131072, "experts": 256, "k": 8, "normalise": True},
    ]


def _size(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["head", "distill", "router"])
    if op == "head":
        classes, dim = _size(rng, 500, 131072), _size(rng, 32, 4096)
        most = min((1 << 40) // (classes * dim), (1 << 29) // classes)
        return {"op": op, "rows": _size(rng, 16, max(16, min(32768, most))), "dim": dim, "classes": classes,
                "train": rng.random() < 0.75}
    if op == "distill":
        classes = _size(rng, 500, 131072)
        return {"op": op, "rows": _size(rng, 16, max(16, min(32768, (1 << 29) // classes))), "classes": classes,
                "k": _size(rng, 1, 256), "temperature": rng.choice([1.0, 1.5, 2.0, 4.0])}
    experts = _size(rng, 4, 512)
    return {"op": op, "rows": _size(rng, 16, (1 << 25) // experts), "experts": experts,
            "k": _size(rng, 1, min(16, experts)), "normalise": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(shape, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g)

    def uniform(shape):
        return torch.empty(shape, device="cuda").uniform_(0.0, 1.0, generator=g)

    rows = case["rows"]
    if case["op"] == "head":
        # logits of standard deviation 2; one row in twenty is padding
        labels = torch.randint(0, case["classes"], (rows,), device="cuda", generator=g, dtype=torch.int32)
        return {"x": normal((rows, case["dim"])), "w": normal((case["classes"], case["dim"]), 2.0 / math.sqrt(case["dim"])),
                "labels": torch.where(uniform((rows,)) < 0.05, -100, labels), "ug": torch.ones(1, device="cuda")}
    if case["op"] == "distill":
        classes, k = case["classes"], case["k"]
        # k classes of each row, no two alike, in the order of the teacher's falling logits
        span = classes // k
        ids = (uniform((rows, k)) * span).to(torch.int32).clamp(max=span - 1)
        ids = ids + span * torch.argsort(uniform((rows, k)), dim=1).to(torch.int32)
        # one row in twenty is padding, one in ten has entries for half of its places
        kind, place = uniform((rows, 1)), torch.arange(k, device="cuda")
        ids = torch.where((kind < 0.05) | ((kind > 0.9) & (place >= (k + 1) // 2)), -1, ids)
        return {"x": normal((rows, classes), 2.0), "ids": ids, "teacher": torch.sort(normal((rows, k), 2.0) + 6.0, dim=1, descending=True)[0],
                "ug": torch.ones(1, device="cuda")}
    return {"x": normal((rows, case["experts"]), 1.5), "keep": (uniform((rows,)) >= 0.05).to(torch.int32),
            "gw": normal((rows, case["k"])), "ug": torch.full((1,), 0.01, device="cuda")}


class _State:
    """A case's inputs (.t) and the buffers that its results go to (.o)."""


def prepare(case, seed):
    s = _State()
    s.case, s.t = case, _inputs(case, seed)
    rows = case["rows"]

    def floats(*shape):
        return torch.zeros(shape, device="cuda")

    if case["op"] == "head":
        s.o = {"loss": floats(1), "row_lse": floats(rows)}
        if case["train"]:
            s.o.update(grad_x=floats(rows, case["dim"]), grad_w=floats(case["classes"], case["dim"]))
        else:
            s.o["row_loss"] = floats(rows)
    elif case["op"] == "distill":
        s.o = {"loss": floats(1), "row_lse": floats(rows), "grad_x": floats(rows, case["classes"])}
    else:
        s.o = {"weights": floats(rows, case["k"]), "loss": floats(1), "grad_x": floats(rows, case["experts"]),
               "chosen": torch.zeros((rows, case["k"]), device="cuda", dtype=torch.int32),
               "counts": torch.zeros(case["experts"], device="cuda", dtype=torch.int32)}
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------------------
# one pass: the plain forms
# ---------------------------------------------------------------------------------------
def _plain_head(t, train):
    x, w, keep = t["x"], t["w"], t["labels"] >= 0
    place = t["labels"].clamp(min=0).long().unsqueeze(1)
    n = keep.sum().clamp(min=1)
    z = x @ w.t()
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(1)
    row = torch.where(keep, lse - z.gather(1, place).squeeze(1), 0.0)
    out = {"loss": (row.sum() / n).reshape(1), "row_lse": torch.where(keep, lse, 0.0)}
    if not train:
        return dict(out, row_loss=row)
    c = torch.where(keep, t["ug"] / n, 0.0).unsqueeze(1)
    g = e * (c / total)
    g.scatter_add_(1, place, -c)
    return dict(out, grad_x=g @ w, grad_w=g.t() @ x)


def _plain_distill(t, temperature):
    x, ids = t["x"], t["ids"]
    there = ids >= 0
    keep = there.any(1, keepdim=True)
    n = keep.sum().clamp(min=1)
    place = ids.clamp(min=0).long()
    y = x / temperature
    top = y.amax(1, keepdim=True)
    e = torch.exp(y - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    u = torch.where(there, t["teacher"] / temperature, -math.inf)
    best = torch.where(keep, u.amax(1, keepdim=True), 0.0)
    v = torch.where(there, torch.exp(u - best), 0.0)
    mass = torch.where(keep, v.sum(1, keepdim=True), 1.0)
    q = v / mass
    part = q * (torch.where(there, u, 0.0) - best - torch.log(mass) - (y.gather(1, place) - lse))
    loss = torch.where(there, part, 0.0).sum() * (temperature * temperature) / n
    c = torch.where(keep, t["ug"] * temperature / n, 0.0)
    g = e * (c / total)
    g.scatter_add_(1, place, -q * c)
    return {"loss": loss.reshape(1), "row_lse": torch.where(keep, lse, 0.0).squeeze(1), "grad_x": g}


def _plain_router(t, k, normalise):
    x, keep = t["x"], (t["keep"] != 0).unsqueeze(1)
    experts = x.shape[1]
    n = keep.sum().clamp(min=1)
    e = torch.exp(x - x.amax(1, keepdim=True))
    p = e / e.sum(1, keepdim=True)
    place = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
    hit = torch.zeros_like(x, dtype=torch.bool).scatter_(1, place, True) & keep
    counts = hit.sum(0)
    f = counts / (n * k)
    loss = experts * (f * (torch.where(keep, p, 0.0).sum(0) / n)).sum()
    picked = p.gather(1, place)
    weights = picked / picked.sum(1, keepdim=True) if normalise else picked
    inner = (t["gw"] * weights).sum(1, keepdim=True)
    g = (t["ug"] * experts / n) * p * (f - (f * p).sum(1, keepdim=True))
    if normalise:
        g.scatter_add_(1, place, weights * (t["gw"] - inner))
    else:
        g = g - p * inner
        g.scatter_add_(1, place, picked * t["gw"])
    return {"weights": torch.where(keep, weights, 0.0), "chosen": torch.where(keep, place, -1).to(torch.int32),
            "counts": counts.to(torch.int32), "loss": loss.reshape(1), "grad_x": torch.where(keep, g, 0.0)}


# ---------------------------------------------------------------------------------------
# one pass: the library's calls
# ---------------------------------------------------------------------------------------
def _library_pass(s):
    global _started
    import mantle_amd as m

    if not _started:  # every call is queued, as in a program that trains for many steps
        m.init(0, asynchronous=True)
        _started = True
    case = s.case
    a = {k: (m.IndexTensor if v.dtype == torch.int32 else m.Tensor).over(v.data_ptr(), tuple(v.shape), v)
         for k, v in (*s.t.items(), *s.o.items())}
    if case["op"] == "head" and case["train"]:
        m.linear_cross_entropy_step(a["loss"], a["grad_x"], a["grad_w"], a["x"], a["w"], a["labels"], a["ug"],
                                    row_lse=a["row_lse"], accumulate=False)
    elif case["op"] == "head":
        m.linear_cross_entropy_forward(a["loss"], a["row_lse"], a["x"], a["w"], a["labels"], row_loss=a["row_loss"])
    elif case["op"] == "distill":
        m.distill_step(a["loss"], a["grad_x"], a["x"], a["ids"], a["teacher"], a["ug"],
                       temperature=case["temperature"], row_lse=a["row_lse"], accumulate=False)
    else:
        m.router_forward(a["weights"], a["chosen"], a["counts"], a["loss"], a["x"], keep=a["keep"],
                         normalise=case["normalise"])
        m.router_backward(a["grad_x"], a["x"], a["chosen"], a["counts"], a["gw"], a["ug"], keep=a["keep"],
                          normalise=case["normalise"], accumulate=False)
    return s.o


def run(s):
    if own:
        return _library_pass(s)
    if s.case["op"] == "head":
        return _plain_head(s.t, s.case["train"])
    if s.case["op"] == "distill":
        return _plain_distill(s.t, s.case["temperature"])
    return _plain_router(s.t, s.case["k"], s.case["normalise"])


# ---------------------------------------------------------------------------------------
# the least that a pass moves and computes
# ---------------------------------------------------------------------------------------
def work(case):
    rows = case["rows"]
    if case["op"] == "head":
        dim, classes = case["dim"], case["classes"]
        inputs = 4 * (rows * dim + classes * dim + rows)
        if not case["train"]:
            return {"bytes": inputs + 8 * rows + 4, "flops": 2 * rows * dim * classes + 4 * rows * classes}
        return {"bytes": inputs + 4 * (rows * dim + classes * dim + rows + 1),
                "flops": 6 * rows * dim * classes + 8 * rows * classes}
    if case["op"] == "distill":
        n, k = rows * case["classes"], rows * case["k"]
        return {"bytes": 4 * (2 * n + 2 * k + rows + 1), "flops": 8 * n + 10 * k}
    n, k = rows * case["experts"], rows * case["k"]
    # the logits and padding marks read by both calls; weights, ids and their gradient once over
    return {"bytes": 4 * (3 * n + 2 * rows + 4 * k + 2 * case["experts"] + 1), "flops": 16 * n + 6 * k}


# ---------------------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    t = _inputs(case, seed)
    d = {k: v.double() if v.is_floating_point() else v.long() for k, v in t.items()}
    if case["op"] == "head":
        kept = d["labels"] >= 0
        x, w = d["x"].requires_grad_(case["train"]), d["w"].requires_grad_(case["train"])
        z = torch.nn.functional.linear(x, w)
        lse = torch.logsumexp(z.detach(), 1) * kept
        row = torch.nn.functional.cross_entropy(z, d["labels"], ignore_index=-100, reduction="none")
        loss = row.sum() / max(1, int(kept.sum()))
        out = {"loss": loss.detach().reshape(1), "row_lse": lse}
        if not case["train"]:
            return dict(out, row_loss=row)
        loss.backward()
        return dict(out, grad_x=x.grad, grad_w=w.grad)
    if case["op"] == "distill":
        tau, rows = case["temperature"], case["rows"]
        there = d["ids"] >= 0
        some = there.any(1)
        n = max(1, int(some.sum()))
        x = d["x"].requires_grad_(True)
        logp = torch.log_softmax(x / tau, 1)
        q = torch.softmax(torch.where(there, d["teacher"] / tau, -1e300), 1) * there
        at = torch.arange(rows, device="cuda").unsqueeze(1).expand_as(q)
        loss = tau * tau / n * (torch.special.xlogy(q, q) - q * logp[at, d["ids"].clamp(min=0)]).sum()
        loss.backward(d["ug"][0])
        return {"loss": loss.detach().reshape(1), "row_lse": torch.logsumexp(x.detach() / tau, 1) * some, "grad_x": x.grad}
    k, experts = case["k"], case["experts"]
    kept = d["keep"] != 0
    n = max(1, int(kept.sum()))
    x = d["x"].requires_grad_(True)
    p = torch.softmax(x, 1)
    order = torch.argsort(-t["x"], dim=1, stable=True)[:, :k]
    counts = torch.bincount(order[kept].reshape(-1), minlength=experts)
    weights = torch.softmax(x.gather(1, order), 1) if case["normalise"] else p.gather(1, order)
    weights = weights * kept.unsqueeze(1)
    loss = experts * (counts.double() / (n * k)) @ (p * kept.unsqueeze(1)).sum(0) / n
    (loss * d["ug"][0] + (weights * d["gw"]).sum()).backward()
    return {"weights": weights.detach(), "chosen": torch.where(kept.unsqueeze(1), order, -1).to(torch.int32),
            "counts": counts.to(torch.int32), "loss": loss.detach().reshape(1), "grad_x": x.grad}
