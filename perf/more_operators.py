"""What stands around the losses of a language model, as measurable cases.

Four operators, each in its plain form (torch operations in 32 bits, in 64 where a border decides) and as the
library's calls:

* ``norm``: root-mean-square norm with the residual's addition. ``h = x + residual`` is the residual stream,
  ``out = h / sqrt(mean h^2 + eps) * w`` over the rows of ``[rows, dim]``. A training step returns both, the
  gradient of ``x`` (and of ``residual``, which is the same) from the gradients of both, and that of ``w``.
* ``route``: routing to experts by sigmoid or softmax scores. A bias for balance, which carries no gradient,
  is added to the scores for the choice alone; of ``groups`` of experts those with the largest sums of their two best
  count; of what is left the ``k`` largest are chosen, ties to the lowest index. A pass returns the weights
  (the chosen's own scores, normalised or not, times ``scale``), the choice, each expert's count and the logits' gradient.
* ``clip``: the norm of all gradients of a model, or an Adam step with the gradients scaled to a largest norm.
* ``sample``: a token for each row of logits ``[rows, classes]`` from a uniform number, after temperature, top-k,
  top-p and min-p, each row with its own; and the logarithm of the probability with which it was drawn.

Data is fp32, the library's one type; ids, counts and top-k are int32.
"""
import math
import random

import torch

own = False
_started = False


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------
def listed():
    return [
        # the norm before a layer when one token is generated
        {"name": "norm_token", "op": "norm", "rows": 1, "dim": 4096, "train": False},
        # a ragged micro-batch, and a width that no vector divides
        {"name": "norm_odd", "op": "norm", "rows": 1023, "dim": 513, "train": True},
        # a training step's batch over a wide model
        {"name": "norm_large", "op": "norm", "rows": 16384, "dim": 4096, "train": True},
        # the router of a small model's batch
        {"name": "route_small", "op": "route", "rows": 64, "experts": 16, "k": 2, "groups": 4, "keep_groups": 2,
         "sigmoid": True, "normalise": True, "scale": 1.0},
        # a ragged batch over groups of an odd size, softmax scores as they are
        {"name": "route_odd", "op": "route", "rows": 33333, "experts": 60, "k": 5, "groups": 6, "keep_groups": 3,
         "sigmoid": False, "normalise": False, "scale": 1.0},
        # a large batch over many experts
        {"name": "route_256", "op": "route", "rows": 131072, "experts": 256, "k": 8, "groups": 8, "keep_groups": 4,
         "sigmoid": True, "normalise": True, "scale": 2.5},
        # an optimizer step of a small model
        {"name": "clip_small", "op": "clip", "tensors": 8, "least": 32, "most": 65536, "step": True, "clipped": True},
        # the norm over hundreds of tensors of all sizes
        {"name": "clip_many", "op": "clip", "tensors": 400, "least": 1, "most": 262144, "step": False, "clipped": True},
        # an optimizer step of a model whose tensors are matrices
        {"name": "clip_large", "op": "clip", "tensors": 24, "least": 1 << 20, "most": 1 << 23, "step": True, "clipped": True},
        # the next token of one sequence
        {"name": "sample_one", "op": "sample", "rows": 1, "classes": 32000, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "mixed": False},
        # a few sequences, each with settings of its own, over an odd vocabulary
        {"name": "sample_odd", "op": "sample", "rows": 33, "classes": 30011, "top_k": 50, "top_p": 0.95, "min_p": 0.05, "mixed": True},
        # many sequences at once over a large vocabulary
        {"name": "sample_large", "op": "sample", "rows": 512, "classes": 131072, "top_k": 200, "top_p": 0.95, "min_p": 0.02, "mixed": True},
    ]


def _size(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "route", "clip", "sample"])
    if op == "norm":
        dim = _size(rng, 16, 16384)
        return {"op": op, "rows": _size(rng, 1, min(131072, (1 << 26) // dim)), "dim": dim, "train": rng.random() < 0.7}
    if op == "route":
        groups, each = rng.choice([1, 2, 4, 5, 8, 16]), _size(rng, 2, 64)
        while groups * each > 512:
            each //= 2
        kept = rng.randint((groups + 1) // 2, groups)
        return {"op": op, "rows": _size(rng, 16, (1 << 25) // (groups * each)), "experts": groups * each,
                "k": _size(rng, 1, min(16, kept * each)), "groups": groups, "keep_groups": kept,
                "sigmoid": rng.random() < 0.5, "normalise": rng.random() < 0.5, "scale": rng.choice([1.0, 2.5])}
    if op == "clip":
        tensors = _size(rng, 1, 400)
        most = _size(rng, 64, min(1 << 24, (1 << 26) // tensors))
        return {"op": op, "tensors": tensors, "least": max(1, most // rng.choice([2, 16, 1 << 18])), "most": most,
                "step": rng.random() < 0.6, "clipped": rng.random() < 0.7}
    classes = _size(rng, 500, 131072)
    return {"op": op, "rows": _size(rng, 1, min(4096, (1 << 26) // classes)), "classes": classes,
            "top_k": rng.choice([0, 1, 20, 50, 1000]), "top_p": rng.choice([1.0, 0.95, 0.8, 0.5]),
            "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]), "mixed": rng.random() < 0.6}


def _tensor_sizes(case):
    """The tensors' sizes of a model, which go with the case and not with the seed."""
    r = random.Random(case["tensors"] * 1000003 + case["most"])
    return [_size(r, case["least"], case["most"]) for _ in range(case["tensors"])]


# ---------------------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------------------
_EPS = 1e-5  # of the norm
_LR, _BETA1, _BETA2, _ADAM_EPS, _MAX_NORM, _STEPS = 1e-3, 0.9, 0.999, 1e-8, 1.0, 9


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(shape, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g)

    def uniform(shape, lo=0.0, hi=1.0):
        return torch.empty(shape, device="cuda").uniform_(lo, hi, generator=g)

    def pick(rows, *values):
        at = torch.randint(0, len(values), (rows,), device="cuda", generator=g)
        return torch.tensor(values, device="cuda")[at]

    if case["op"] == "norm":
        size = (case["rows"], case["dim"])
        t = {"x": normal(size), "residual": normal(size, 2.0), "w": 1.0 + normal(case["dim"], 0.2)}
        if case["train"]:
            t.update(grad_out=normal(size), grad_sum=normal(size))
        return t
    if case["op"] == "route":
        rows, experts = case["rows"], case["experts"]
        # the bias moves the choice by about as much as the scores differ; one row in twenty is padding
        return {"x": normal((rows, experts), 1.5), "bias": normal(experts, 0.1 if case["sigmoid"] else 0.5 / experts),
                "keep": (uniform(rows) >= 0.05).to(torch.int32), "gw": normal((rows, case["k"]))}
    if case["op"] == "clip":
        # every tensor begins at a multiple of 64 elements of an arena; the norm is about 3, or a third
        sizes = _tensor_sizes(case)
        n = sum((k + 63) // 64 * 64 for k in sizes)
        t = {"g": normal(n, (3.0 if case["clipped"] else 0.3) / math.sqrt(sum(sizes)))}
        if case["step"]:
            std = float(3.0 / math.sqrt(sum(sizes)))
            t.update(p=normal(n, 0.02), m=normal(n, 0.1 * std), v=uniform(n, 0.0, 0.1 * std * std))
        at = 0
        for k in sizes:  # the gaps between tensors hold zeros
            end = (at + k + 63) // 64 * 64
            for a in t.values():
                a[at + k:end] = 0.0
            at = end
        return t
    rows, classes = case["rows"], case["classes"]
    # a bulk of unlikely classes, and a few dozen that stand out
    x = normal((rows, classes), 2.0)
    some = torch.randint(0, classes, (rows, 32), device="cuda", generator=g)
    x.scatter_add_(1, some, uniform((rows, 32), 2.0, 12.0))
    t = {"x": x, "u": uniform(rows)}
    if case["mixed"]:  # one row in five takes the largest
        t.update(temperature=pick(rows, 0.0, 0.5, 0.7, 1.0, 1.3), top_k=pick(rows, 0, case["top_k"]).to(torch.int32),
                 top_p=pick(rows, 1.0, case["top_p"]), min_p=pick(rows, 0.0, case["min_p"]))
    else:
        t.update(temperature=torch.full((rows,), 0.8, device="cuda"),
                 top_k=torch.full((rows,), case["top_k"], device="cuda", dtype=torch.int32),
                 top_p=torch.full((rows,), case["top_p"], device="cuda"), min_p=torch.full((rows,), case["min_p"], device="cuda"))
    return t


def _slices(case, arena):
    at, out = 0, []
    for k in _tensor_sizes(case):
        out.append(arena[at:at + k])
        at += (k + 63) // 64 * 64
    return out


class _State:
    """A case's inputs (.t), the buffers that its results go to (.o), the steps taken so far, and with the library
    its tensors over both (.a) and its optimizer."""


def prepare(case, seed):
    s = _State()
    s.case, s.t, s.steps = case, _inputs(case, seed), _STEPS

    def floats(*shape):
        return torch.zeros(shape, device="cuda")

    def ids(*shape):
        return torch.zeros(shape, device="cuda", dtype=torch.int32)

    if case["op"] == "norm":
        size = (case["rows"], case["dim"])
        s.o = {"out": floats(*size), "sum": floats(*size)}
        if case["train"]:
            s.o.update(grad_x=floats(*size), grad_w=floats(case["dim"]))
    elif case["op"] == "route":
        rows, k = case["rows"], case["k"]
        s.o = {"weights": floats(rows, k), "chosen": ids(rows, k), "counts": ids(case["experts"]),
               "grad_x": floats(rows, case["experts"])}
    elif case["op"] == "clip":
        s.o = {"norm": floats(1)}
    else:
        s.o = {"token": ids(case["rows"]), "logprob": floats(case["rows"])}
    if own:
        _library_state(s)
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------------------
# one pass: the plain forms
# ---------------------------------------------------------------------------------------
def _plain_norm(t, train):
    h = t["x"] + t["residual"]
    scale = torch.rsqrt((h * h).mean(1, keepdim=True) + _EPS)
    unit = h * scale
    out = {"out": unit * t["w"], "sum": h}
    if not train:
        return out
    g = t["grad_out"] * t["w"]
    grad_x = t["grad_sum"] + scale * (g - unit * (g * unit).mean(1, keepdim=True))
    return dict(out, grad_x=grad_x, grad_w=(t["grad_out"] * unit).sum(0))


def _plain_route(t, case):
    x, keep = t["x"].double(), (t["keep"] != 0).unsqueeze(1)
    rows, experts = x.shape
    k, groups = case["k"], case["groups"]
    if case["sigmoid"]:
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        e = torch.exp(x - x.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    biased = score + t["bias"].double()
    if groups > 1:
        best = torch.sort(biased.view(rows, groups, -1), dim=2, descending=True)[0][:, :, :2].sum(2)
        order = torch.sort(best, dim=1, descending=True, stable=True)[1][:, :case["keep_groups"]]
        open_ = torch.zeros((rows, groups), device=x.device, dtype=torch.bool).scatter_(1, order, True)
        biased = torch.where(open_.repeat_interleave(experts // groups, 1), biased, -math.inf)
    place = torch.sort(biased, dim=1, descending=True, stable=True)[1][:, :k]
    hit = torch.zeros_like(x, dtype=torch.bool).scatter_(1, place, True) & keep
    picked = score.gather(1, place).float()
    total = picked.sum(1, keepdim=True) if case["normalise"] else torch.ones_like(picked[:, :1])
    share = picked / total
    gw = t["gw"] * case["scale"]
    inner = (gw * share).sum(1, keepdim=True)
    grad = torch.zeros_like(t["x"])
    if case["sigmoid"]:
        # share is s / total: its gradient by the logits passes s (1 - s)
        rest = (1.0 / (1.0 + torch.exp(x.gather(1, place)))).float()
        grad.scatter_add_(1, place, share * rest * ((gw - inner) if case["normalise"] else gw))
    elif case["normalise"]:
        grad.scatter_add_(1, place, share * (gw - inner))
    else:
        grad = -score.float() * inner
        grad.scatter_add_(1, place, picked * gw)
    return {"weights": torch.where(keep, share * case["scale"], 0.0), "chosen": torch.where(keep, place, -1).to(torch.int32),
            "counts": hit.sum(0).to(torch.int32), "grad_x": torch.where(keep, grad, 0.0)}


def _power(b, n):
    """b ** n with every product rounded to 32 bits."""
    a, r = torch.tensor(b, dtype=torch.float32), torch.tensor(1.0, dtype=torch.float32)
    while n:
        if n & 1:
            r = r * a
        a, n = a * a, n >> 1
    return float(r)


def _plain_clip(s):
    grads = _slices(s.case, s.t["g"])
    total = torch.zeros((), device="cuda", dtype=torch.float64)
    for g in grads:
        total += g.double().square().sum()
    norm = torch.sqrt(total)
    out = {"norm": norm.float().reshape(1)}
    if not s.case["step"]:
        return out
    s.steps += 1
    c = torch.clamp(_MAX_NORM / norm, max=1.0).float()
    f32 = torch.tensor([_BETA1, _BETA2], dtype=torch.float32)
    b1, b2 = (float(v) for v in f32)
    c1, c2 = (float(v) for v in 1.0 - f32)
    d1 = float(torch.tensor(1.0) - _power(_BETA1, s.steps))
    d2 = float(torch.tensor(1.0) - _power(_BETA2, s.steps))
    for p, g, m, v in zip(*(_slices(s.case, s.t[a]) for a in ("p", "g", "m", "v"))):
        g = g * c
        m.copy_(b1 * m + c1 * g)
        v.copy_(b2 * v + c2 * g * g)
        p.copy_(p - _LR * ((m / d1) / (torch.sqrt(v / d2) + _ADAM_EPS)))
    return dict(out, p=s.t["p"], m=s.t["m"], v=s.t["v"])


def _plain_sample(t):
    x = t["x"]
    rows, classes = x.shape
    greedy = t["temperature"] <= 0
    heat = torch.where(greedy, 1.0, t["temperature"]).double().unsqueeze(1)
    k = torch.where(t["top_k"] <= 0, classes, t["top_k"]).clamp(max=classes)
    k = torch.where(greedy, 1, k).unsqueeze(1)
    value, order = torch.sort(x, dim=1, descending=True, stable=True)
    e = torch.exp((value.double() - value[:, :1].double()) / heat)
    e = torch.where(torch.arange(classes, device=x.device) < k, e, 0.0)
    before = torch.cumsum(e, 1) - e
    fits = before < t["top_p"].double().unsqueeze(1) * e.sum(1, keepdim=True)
    fits[:, 0] = True
    e = torch.where(fits & (e >= t["min_p"].double().unsqueeze(1)), e, 0.0)
    mass = torch.zeros_like(e).scatter_(1, order, e)
    total = mass.sum(1, keepdim=True)
    token = (torch.cumsum(mass, 1) <= t["u"].double().unsqueeze(1) * total).sum(1).clamp(max=classes - 1)
    drawn = mass.gather(1, token.unsqueeze(1))
    return {"token": token.to(torch.int32), "logprob": torch.log(drawn / total).squeeze(1).float()}


# ---------------------------------------------------------------------------------------
# one pass: the library's calls
# ---------------------------------------------------------------------------------------
def _library_state(s):
    global _started
    import mantle_amd as m

    if not _started:  # every call is queued, as in a program that trains for many steps
        m.init(0, asynchronous=True)
        _started = True

    def over(v):
        return (m.IndexTensor if v.dtype == torch.int32 else m.Tensor).over(v.data_ptr(), tuple(v.shape), v)

    s.a = {k: over(v) for k, v in (*s.t.items(), *s.o.items())}
    if s.case["op"] == "clip":
        each = {k: [over(v) for v in _slices(s.case, s.t[k])] for k in s.t}
        s.grads = each["g"]
        if s.case["step"]:
            s.adam = m.Adam(list(zip(each["p"], each["g"])), lr=_LR, beta1=_BETA1, beta2=_BETA2, epsilon=_ADAM_EPS, max_norm=_MAX_NORM)
            s.adam.momentum_grads[:], s.adam.rms_grads[:] = each["m"], each["v"]
            s.adam.grad_norm, s.adam.iter = s.a["norm"], _STEPS


def _library_pass(s):
    import mantle_amd as m

    case, a = s.case, s.a
    if case["op"] == "norm":
        m.rms_norm_forward(a["out"], a["x"], a["w"], residual=a["residual"], sum=a["sum"], eps=_EPS)
        if case["train"]:
            m.rms_norm_backward(a["grad_x"], a["grad_w"], a["grad_out"], a["sum"], a["w"], grad_sum=a["grad_sum"], eps=_EPS,
                                accumulate=False)
    elif case["op"] == "route":
        scores = "sigmoid" if case["sigmoid"] else "softmax"
        m.group_router_forward(a["weights"], a["chosen"], a["counts"], a["x"], bias=a["bias"], keep=a["keep"],
                               groups=case["groups"], keep_groups=case["keep_groups"], scores=scores,
                               normalise=case["normalise"], scale=case["scale"])
        m.group_router_backward(a["grad_x"], a["x"], a["chosen"], a["gw"], keep=a["keep"], scores=scores,
                                normalise=case["normalise"], scale=case["scale"], accumulate=False)
    elif case["op"] == "clip":
        if not case["step"]:
            m.grad_norm(a["norm"], s.grads)
            return s.o
        s.adam.step()
        return dict(s.o, p=s.t["p"], m=s.t["m"], v=s.t["v"])
    else:
        m.sample_tokens(a["token"], a["x"], a["u"], temperature=a["temperature"], top_k=a["top_k"], top_p=a["top_p"],
                        min_p=a["min_p"], logprob=a["logprob"])
    return s.o


def run(s):
    if own:
        return _library_pass(s)
    if s.case["op"] == "norm":
        return _plain_norm(s.t, s.case["train"])
    if s.case["op"] == "route":
        return _plain_route(s.t, s.case)
    if s.case["op"] == "clip":
        return _plain_clip(s)
    return _plain_sample(s.t)


# ---------------------------------------------------------------------------------------
# the least that a pass moves and computes
# ---------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        n, dim = case["rows"] * case["dim"], case["dim"]
        if not case["train"]:
            return {"bytes": 4 * (4 * n + dim), "flops": 5 * n}
        # x, residual, both gradients; sum, out and the gradients of x and w
        return {"bytes": 4 * (7 * n + 2 * dim), "flops": 15 * n}
    if case["op"] == "route":
        n, k = case["rows"] * case["experts"], case["rows"] * case["k"]
        return {"bytes": 4 * (2 * n + case["rows"] + 3 * k + 2 * case["experts"]), "flops": 12 * n + 8 * k}
    if case["op"] == "clip":
        n = sum(_tensor_sizes(case))
        return {"bytes": (28 if case["step"] else 4) * n + 4, "flops": (18 if case["step"] else 2) * n}
    n = case["rows"] * case["classes"]
    return {"bytes": 4 * (n + 7 * case["rows"]), "flops": 6 * n}


# ---------------------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    t = _inputs(case, seed)
    d = {k: v.double() if v.is_floating_point() else v.long() for k, v in t.items()}
    if case["op"] == "norm":
        h = (d["x"] + d["residual"]).requires_grad_(case["train"])
        w = d["w"].requires_grad_(case["train"])
        out = h / torch.sqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / case["dim"] + _EPS) * w
        got = {"out": out.detach(), "sum": h.detach()}
        if case["train"]:
            ((out * d["grad_out"]).sum() + (h * d["grad_sum"]).sum()).backward()
            got.update(grad_x=h.grad, grad_w=w.grad)
        return got
    if case["op"] == "route":
        rows, experts, k = case["rows"], case["experts"], case["k"]
        kept = d["keep"] != 0
        x = d["x"].requires_grad_(True)
        score = torch.sigmoid(x) if case["sigmoid"] else torch.softmax(x, 1)
        rank = (score + d["bias"]).detach()
        each = experts // case["groups"]
        if case["groups"] > 1:
            two = torch.topk(rank.reshape(-1, each), min(2, each))[0].sum(1).reshape(rows, -1)
            shut = torch.argsort(-two, dim=1, stable=True)[:, case["keep_groups"]:]
            at = (shut.unsqueeze(2) * each + torch.arange(each, device="cuda")).reshape(rows, -1)
            rank = rank.scatter(1, at, -math.inf)
        order = torch.argsort(-rank, dim=1, stable=True)[:, :k]
        w = score.gather(1, order)
        if case["normalise"]:
            w = w / w.sum(1, keepdim=True)
        w = case["scale"] * w * kept.unsqueeze(1)
        (w * d["gw"]).sum().backward()
        return {"weights": w.detach(), "chosen": torch.where(kept.unsqueeze(1), order, -1).to(torch.int32),
                "counts": torch.bincount(order[kept].reshape(-1), minlength=experts).to(torch.int32), "grad_x": x.grad}
    if case["op"] == "clip":
        # the gaps of the arenas hold zeros, which change no norm and stay as they are
        norm = torch.linalg.vector_norm(d["g"])
        out = {"norm": norm.reshape(1)}
        if case["step"]:
            b1, b2, lr, eps = (float(v) for v in torch.tensor([_BETA1, _BETA2, _LR, _ADAM_EPS], dtype=torch.float32))
            g = d["g"] * min(1.0, _MAX_NORM / float(norm))
            m = torch.lerp(g, d["m"], b1)
            v = torch.lerp(g * g, d["v"], b2)
            rate = torch.sqrt(v / (1.0 - b2 ** (_STEPS + 1))) + eps
            out.update(p=d["p"] - lr / (1.0 - b1 ** (_STEPS + 1)) * m / rate, m=m, v=v)
        return out
    rows, classes = case["rows"], case["classes"]
    token, logprob = [], []
    for r in range(rows):
        x, heat, k = d["x"][r], float(d["temperature"][r]), int(d["top_k"][r])
        if heat <= 0:
            token.append(torch.argmax(x))
            logprob.append(torch.zeros((), device="cuda", dtype=torch.float64))
            continue
        # the classes from the likeliest on, cut by each of the three
        order = torch.argsort(-x, stable=True)[:k if k > 0 else classes]
        p = torch.softmax(x[order] / heat, 0)
        many = int(torch.searchsorted(torch.cumsum(p, 0), d["top_p"][r])) + 1 if float(d["top_p"][r]) < 1 else len(order)
        many = max(1, min(many, int((p / p[0] >= d["min_p"][r]).sum())))
        order = torch.sort(order[:many])[0]
        p = torch.softmax(x[order] / heat, 0)
        at = torch.searchsorted(torch.cumsum(p, 0), d["u"][r], right=True).clamp(max=many - 1)
        token.append(order[at])
        logprob.append(torch.log(p[at]))
    return {"token": torch.stack(token).to(torch.int32), "logprob": torch.stack(logprob)}
